"""Drafted-token trees over the 4-bit cache, and 8-bit integer products, as timed cases.

Five paths, each in its plain form (elementary torch operations) and, where
``own`` is true, through the entry points a program calls:

* ``tree``   -- attention of the rows of a tree of drafted tokens, which are at
  the end of the cache: a row sees all slots before the tree, and of the tree
  the rows its mask names (``DeviceOps.kv4_tree_attention``);
* ``accept`` -- the drafted tokens that the target's greedy choice confirms,
  from the logits of the tree's rows (``tree_accept``);
* ``keep``   -- a tree's keys and values written (``kv4_append``), the accepted
  ones moved together (``kv4_keep``), and these read back (``kv4_read``);
* ``w8``     -- products with 8-bit integer weights, a scale for each token
  and each output channel (``w8_matmul``);
* ``gated``  -- both projections of a feed-forward block, the activation and
  the product in one call, in the same number format (``w8_gated``).

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

8-bit numbers: a token's scale is s = f32(max |x| / 127) and its codes are the
integers nearest x / s (ties to even); a weight row has int8 codes and an f32
scale of its own; y = s_token s_row sum(codes codes).
"""
import math
import random

import torch

own = False

PAGE = 64
BITS = (6, 22, 2, 18, 14, 30, 10, 26)
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_CODE = {"f32": 0, "f16": 1, "bf16": 2}
ACTIVATIONS = {"silu": 0, "gelu": 1}


def listed():
    return [
        # A small tree (8 drafted tokens) of an 8B decoder's heads, early in a conversation.
        {"name": "tree_t1_8", "path": "tree", "type": "f32", "seqs": 1, "rows_lo": 8, "rows": 8, "len_lo": 777,
         "len": 777, "heads": 32, "kv": 8, "dim": 128, "window": 0},
        # A tree of 60 behind a long document, eight queries to a kv head.
        {"name": "tree_t1_60_long", "path": "tree", "type": "bf16", "seqs": 1, "rows_lo": 60, "rows": 60,
         "len_lo": 32001, "len": 32001, "heads": 64, "kv": 8, "dim": 128, "window": 0},
        # 16 lanes with trees of 5 to 26 drafted tokens behind 500 to 8000 slots.
        {"name": "tree_b16", "path": "tree", "type": "bf16", "seqs": 16, "rows_lo": 5, "rows": 26, "len_lo": 500,
         "len": 8000, "heads": 32, "kv": 8, "dim": 128, "window": 0},
        # The choice along one tree, f32 logits.
        {"name": "accept_t1_8", "path": "accept", "type": "f32", "seqs": 1, "rows_lo": 8, "rows": 8, "vocab": 128256},
        # The choice of 16 lanes, bf16 logits of a wide vocabulary.
        {"name": "accept_b16", "path": "accept", "type": "bf16", "seqs": 16, "rows_lo": 5, "rows": 26,
         "vocab": 151936},
        # One lane commits what was accepted of 8.
        {"name": "keep_t1_8", "path": "keep", "type": "f32", "seqs": 1, "rows_lo": 8, "rows": 8, "len_lo": 777,
         "len": 777, "kv": 8, "dim": 128},
        # 32 lanes do.
        {"name": "keep_b32", "path": "keep", "type": "bf16", "seqs": 32, "rows_lo": 5, "rows": 26, "len_lo": 500,
         "len": 8000, "kv": 8, "dim": 128},
        # The attention output projection of one token.
        {"name": "w8_t1_4096x4096", "path": "w8", "type": "f32", "tokens": 1, "in": 4096, "out": 4096},
        # The down projection for a tree of 60.
        {"name": "w8_t60_4096x14336", "path": "w8", "type": "bf16", "tokens": 60, "in": 14336, "out": 4096},
        # A feed-forward projection of a prompt of odd length.
        {"name": "w8_t4001_14336x4096", "path": "w8", "type": "bf16", "tokens": 4001, "in": 4096, "out": 14336},
        # The gated block of one token.
        {"name": "gated_t1_14336x4096", "path": "gated", "type": "f32", "tokens": 1, "in": 4096, "out": 14336,
         "act": "silu"},
        # The gated block of a prompt.
        {"name": "gated_t2001_14336x4096", "path": "gated", "type": "bf16", "tokens": 2001, "in": 4096, "out": 14336,
         "act": "silu"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    path = rng.choice(["tree", "tree", "tree", "accept", "keep", "w8", "w8", "w8", "gated", "gated"])
    ty = rng.choice(["f32", "bf16", "bf16", "f16"])
    if path in ("w8", "gated"):
        # Widths of whole weight blocks (32) mostly, and any others.
        step = rng.choice([32, 32, 32, 1])
        n_in = max(step, _log_int(rng, 64, 14336) // step * step)
        n_out = max(step, min(_log_int(rng, 64, 28672), 14336 * 8192 // n_in) // step * step)
        top = (1 if path == "w8" else 0.5) * 4001 * 4096 * 14336 / (n_in * n_out)
        c = {"path": path, "type": ty, "tokens": _log_int(rng, 1, max(1, min(4097, top))), "in": n_in, "out": n_out}
        if path == "gated":
            c["act"] = rng.choice(sorted(ACTIVATIONS))
        return c
    seqs = _log_int(rng, 1, 64)
    rows = _log_int(rng, 1, 100)
    rows_lo = rng.randint(1, rows)
    if path == "accept":
        vocab = _log_int(rng, 1000, 151936)
        rows = max(1, min(rows, 400 * 151936 // (vocab * seqs)))
        return {"path": path, "type": ty, "seqs": seqs, "rows_lo": min(rows_lo, rows), "rows": rows, "vocab": vocab}
    kv, dim = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128, 256])
    if path == "keep":
        top = 64 * 2000 * 8 * 128 // (seqs * kv * dim)
        n = rows + _log_int(rng, 1, max(1, min(top, 16000)))
        return {"path": path, "type": ty, "seqs": seqs, "rows_lo": rows_lo, "rows": rows,
                "len_lo": rng.randint(1, n), "len": n, "kv": kv, "dim": dim}
    heads = kv * rng.choice([1, 2, 4, 4, 8])
    top = min(60e9 / (4 * rows * heads * dim * seqs), 16 * 8000 * 8 * 128 / (seqs * kv * dim), 64000)
    n = rows + _log_int(rng, 1, max(1, top))
    return {"path": path, "type": ty, "seqs": seqs, "rows_lo": rows_lo, "rows": rows, "len_lo": rng.randint(1, n),
            "len": n, "heads": heads, "kv": kv, "dim": dim, "window": rng.choice([0, 0, 0, 1000])}


# ---- sizes that follow from a case -----------------------------------------

def _spread(lo, hi, n):
    """n whole numbers from hi down to lo."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _rows(c):
    return _spread(c["rows_lo"], c["rows"], c["seqs"])


def _lens(c):
    """Cache lengths with the trees' rows; long trees need not be behind long caches."""
    lens = _spread(c["len_lo"], c["len"], c["seqs"])
    return [max(n, r) for n, r in zip(lens[1::2] + lens[0::2], _rows(c))]


def _kept_rows(c):
    """How many rows each sequence keeps: the last sure token and up to six more."""
    return [min(r, 1 + (3 * i + 2) % 7) for i, r in enumerate(_rows(c))]


def _words(c):
    return -(-c["rows"] // 32)


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


def _trees(seed, rows):
    """Parents of every sequence's rows: row 0 is the last token that is sure,
    the others are drafted, each behind its parent."""
    rng = random.Random(seed)
    return [[-1] + [max(0, i - rng.choice([1, 1, 2, 3, 5, 8])) for i in range(1, n)] for n in rows]


def _ancestors(parents):
    """Per row the set (as an int's bits) of its ancestors and itself."""
    bits = []
    for i, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | (1 << i))
    return bits


def _random_pages(g, n, kv, dim):
    """n pages of keys and values that are roughly N(0, 1): uint8 [n][kv][80 dim]."""
    page = torch.empty(n, kv, 80 * dim, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (kv * 64 * dim))
    for i in range(0, n, step):
        m = min(step, n - i)
        q = (_randn(g, m, kv, 64 * dim, 2) * 2.8 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
        page[i:i + m, :, :64 * dim] = q[..., 0] | (q[..., 1] << 4)
    # Scales of 7 significant bits around 1/2.8, minima around -7.5 of them.
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


def _weights(g, n_out, n_in):
    """int8 codes [out][in] and f32 scales [out]; values of about 1 / sqrt(in)."""
    q = torch.empty(n_out, n_in, dtype=torch.int8, device="cuda")
    step = max(1, (1 << 25) // n_in)
    for i in range(0, n_out, step):
        m = min(step, n_out - i)
        q[i:i + m] = (30 * _randn(g, m, n_in)).round_().clamp_(-127, 127).to(torch.int8)
    return q, torch.exp(0.3 * _randn(g, n_out)) / (30 * math.sqrt(n_in))


def prepare(case, seed):
    c, g = case, _generator(seed)
    ty = TYPES[c["type"]]
    st = {"case": c}
    if c["path"] in ("w8", "gated"):
        # Some channels are far larger than the others, as in trained models.
        size = torch.exp(0.5 * _randn(g, c["in"])) * (1 + 9 * (torch.rand(c["in"], device="cuda", generator=g) < 0.003))
        st.update(x=(_randn(g, c["tokens"], c["in"]) * size).to(ty),
                  y=torch.empty(c["tokens"], c["out"], dtype=ty, device="cuda"))
        for name in (("w",) if c["path"] == "w8" else ("gate", "up")):
            st[name], st[name + "_scale"] = _weights(g, c["out"], c["in"])
        if own:
            _packed(st)
        return st
    rows = _rows(c)
    n, trees = sum(rows), _trees(seed, rows)
    st.update(start=_starts(rows), rows=rows, n=n, max_rows=max(rows), parent=_ints([p for t in trees for p in t]))
    if c["path"] == "accept":
        logits = (2 * _randn(g, n, c["vocab"])).to(ty)
        # A drafted token is right in about two of three places: it is then
        # what its parent's row says.
        says = logits.float().argmax(1)
        up = _ints([s + max(p, 0) for s, t in zip(st["start"].tolist(), trees) for p in t]).long()
        guess = torch.randint(0, c["vocab"], (n,), device="cuda", generator=g)
        right = torch.rand(n, device="cuda", generator=g) < 0.66
        st.update(logits=logits, token=torch.where(right, says[up], guess).to(torch.int32),
                  len=_ints([r + 100 * i for i, r in enumerate(rows)]))
        for name, size in (("path", n), ("count", c["seqs"]), ("next", c["seqs"]), ("new_len", c["seqs"])):
            st[name] = torch.empty(size, dtype=torch.int32, device="cuda")
        return st
    lens, kv, dim = _lens(c), c["kv"], c["dim"]
    width = max(-(-m // PAGE) for m in lens)
    pool = c["seqs"] * width + 7
    st.update(len=_ints(lens), lens=lens, table=_table(g, c["seqs"], width, pool), pages=_random_pages(g, pool, kv, dim))
    if c["path"] == "keep":
        k = _randn(g, n, kv, dim) * torch.exp(0.7 * _randn(g, kv, dim)) + _randn(g, kv, dim)
        rng, count, path = random.Random(seed + 1), _kept_rows(c), []
        for r, m in zip(rows, count):  # a path from row 0 on, padded with -1
            path += [0] + sorted(rng.sample(range(1, r), m - 1)) + [-1] * (r - m)
        kept = sum(count)
        st.update(k=k.to(ty), v=_randn(g, n, kv, dim).to(ty), path=_ints(path), count=_ints(count), kept=kept,
                  kept_start=_starts(count), new_len=_ints([m - r + a for m, r, a in zip(lens, rows, count)]),
                  k_out=torch.empty(kept, kv, dim, dtype=ty, device="cuda"),
                  v_out=torch.empty(kept, kv, dim, dtype=ty, device="cuda"))
        return st
    words, mask = _words(c), []
    for t in trees:
        for bits in _ancestors(t):
            mask += [(bits >> (32 * w)) & 0xFFFFFFFF for w in range(words)]
    mask = [m - (1 << 32) if m >> 31 else m for m in mask]
    # Queries long enough for scores of standard deviation 2.
    st.update(mask=_ints(mask).view(n, words), q=(2.0 * _randn(g, n, c["heads"], dim)).to(ty),
              out=torch.empty(n, c["heads"], dim, dtype=ty, device="cuda"), lse=torch.empty(n, c["heads"], device="cuda"))
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


def _plain_tree(st):
    c = st["case"]
    seqs, kv, dim, top_rows = c["seqs"], c["kv"], c["dim"], st["max_rows"]
    q, real, rows = _row_of(st, st["q"].float())
    group = c["heads"] // kv
    q = q.view(seqs, -1, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, dim)
    s = torch.matmul(q / math.sqrt(dim), _gathered(st, _plain_keys).transpose(2, 3).contiguous())
    slot = torch.arange(s.shape[-1], device="cuda")
    base = st["len"] - rows
    mask, _, _ = _row_of(st, st["mask"])  # [seqs][rows][words]
    bit = torch.arange(top_rows, device="cuda")
    told = ((mask[..., bit // 32] >> (bit % 32)) & 1).bool() & (bit < rows[:, None, None])  # [seqs][rows][rows]
    own_slot = (slot - base[:, None]).clamp(0, top_rows - 1).long()  # [seqs][slots]
    see = torch.gather(told, 2, own_slot[:, None].expand(-1, top_rows, -1))
    see &= (slot < st["len"][:, None])[:, None]
    before = (slot < base[:, None])[:, None].expand_as(see)
    if c["window"]:
        before = before & (slot >= (base[:, None] - c["window"] + told.sum(2))[..., None])
    see = torch.where((slot < base[:, None])[:, None], before, see) & real[..., None]
    s = s.view(seqs, kv, group, top_rows, -1).masked_fill_(~see[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), _gathered(st, _plain_values)).view(*p.shape[:4], dim)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    flat = [x.movedim(3, 1).flatten(2, 3)[real] for x in (o, torch.log(total) + top)]
    return [flat[0].to(TYPES[c["type"]]), flat[1][..., 0]]


def _plain_accept(st):
    c, n = st["case"], st["n"]
    says = st["logits"].float().argmax(1)
    rows = st["start"][1:] - st["start"][:-1]
    first = st["start"][:-1].long()
    i = torch.arange(n, device="cuda")
    inside = torch.repeat_interleave(torch.arange(c["seqs"], device="cuda"), rows.long())
    number = i - first[inside]
    at = torch.zeros(c["seqs"], dtype=torch.long, device="cuda")
    alive = rows > 0
    path = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    count = torch.zeros(c["seqs"], dtype=torch.long, device="cuda")
    said = torch.full((c["seqs"],), -1, dtype=torch.long, device="cuda")
    for _ in range(st["max_rows"]):
        spot = torch.where(alive, first + count, n)  # n: nowhere
        path = torch.cat([path, path.new_zeros(1)]).index_copy_(0, spot, at.to(torch.int32))[:n]
        count = count + alive
        said = torch.where(alive, says[(first + at).clamp(max=n - 1)], said)
        fits = (st["parent"] == at[inside]) & (st["token"] == said[inside]) & (number > at[inside]) & alive[inside]
        child = torch.full((c["seqs"],), n, dtype=torch.long, device="cuda")
        child = child.scatter_reduce(0, inside, torch.where(fits, number, n), "amin")
        alive = child < n
        at = torch.where(alive, child, at)
    new_len = st["len"] - rows + count
    return [path, count.to(torch.int32), said.to(torch.int32), new_len.to(torch.int32)]


def _plain_keep(st):
    rows = st["start"][1:] - st["start"][:-1]
    i = torch.arange(st["n"], device="cuda")
    inside = torch.repeat_interleave(torch.arange(len(st["rows"]), device="cuda"), rows.long())
    taken = i - st["start"][:-1].long()[inside] < st["count"][inside]
    at = (st["start"][:-1][inside] + st["path"])[taken].long()
    return [_plain_quantised(st[x].float())[at].to(TYPES[st["case"]["type"]]) for x in ("k", "v")]


def _plain_token_codes(x):
    """Scales [tokens][1] f32 and codes (f32 whole numbers); quotients in 64 bits, next to halves they decide."""
    x = x.float()
    s = x.abs().amax(1, keepdim=True) / 127
    q = torch.round(x.double() / torch.where(s > 0, s, torch.ones_like(s)).double())
    return s, q.float()


def _plain_product(s, q, w, w_scale):
    return torch.matmul(q, w.float().t()) * s * w_scale


def _plain_run(st):
    c = st["case"]
    if c["path"] == "tree":
        return _plain_tree(st)
    if c["path"] == "accept":
        return _plain_accept(st)
    if c["path"] == "keep":
        return _plain_keep(st)
    s, q = _plain_token_codes(st["x"])
    if c["path"] == "w8":
        return _plain_product(s, q, st["w"], st["w_scale"]).to(TYPES[c["type"]])
    gate = _plain_product(s, q, st["gate"], st["gate_scale"])
    up = _plain_product(s, q, st["up"], st["up_scale"])
    if c["act"] == "silu":
        gate = gate / (1 + torch.exp(-gate))
    else:
        gate = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)))
    return (gate * up).to(TYPES[c["type"]])


# ---- the framework's calls -------------------------------------------------

def _kept(st, name, make):
    """What a program makes once and keeps: handles and workspaces."""
    if name not in st:
        st[name] = make()
    return st[name]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _bytes(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda")


def _packed(st):
    """Weights laid out once, as a program does when it loads a model."""
    import aspida_amd as aa
    c = st["case"]
    dev = _kept(st, "dev", aa.DeviceOps)

    def pack(name):
        p = _bytes(dev.w8_bytes(c["in"], c["out"]))
        dev.w8_pack(st[name].data_ptr(), c["in"], st[name + "_scale"].data_ptr(), c["in"], c["out"], p.data_ptr(),
                    _stream())
        return p
    return [_kept(st, name + "_packed", lambda: pack(name)) for name in ("w", "gate", "up") if name in st]


def _own_run(st):
    import aspida_amd as aa
    c = st["case"]
    sp = _stream()
    dev = _kept(st, "dev", aa.DeviceOps)
    ty = TYPE_CODE[c["type"]]
    if c["path"] in ("w8", "gated"):
        packed = _packed(st)
        work = _kept(st, "work", lambda: _bytes(dev.w8_work_bytes(c["tokens"], c["in"])))
        if c["path"] == "w8":
            dev.w8_matmul(packed[0].data_ptr(), c["in"], c["out"], ty, st["x"].data_ptr(), c["in"], c["tokens"],
                          st["y"].data_ptr(), c["out"], work.data_ptr(), sp)
        else:
            dev.w8_gated(packed[0].data_ptr(), packed[1].data_ptr(), c["in"], c["out"], ACTIVATIONS[c["act"]], ty,
                         st["x"].data_ptr(), c["in"], c["tokens"], st["y"].data_ptr(), c["out"], work.data_ptr(), sp)
        return st["y"]
    n, seqs = st["n"], c["seqs"]
    if c["path"] == "accept":
        work = _kept(st, "work", lambda: _bytes(dev.tree_accept_work_bytes(n, c["vocab"])))
        dev.tree_accept(ty, st["logits"].data_ptr(), c["vocab"], c["vocab"], n, seqs, st["start"].data_ptr(),
                        st["len"].data_ptr(), st["parent"].data_ptr(), st["token"].data_ptr(), st["path"].data_ptr(),
                        st["count"].data_ptr(), st["next"].data_ptr(), st["new_len"].data_ptr(), work.data_ptr(), sp)
        return [st["path"], st["count"], st["next"], st["new_len"]]
    kv, dim = c["kv"], c["dim"]
    cache = _kept(st, "cache", lambda: aa.KV4Cache(dim, kv, st["pages"].shape[0], st["table"].shape[1],
                                                   st["pages"].data_ptr(), st["table"].data_ptr()))
    if c["path"] == "keep":
        row = kv * dim
        dev.kv4_append(cache, ty, st["k"].data_ptr(), row, st["v"].data_ptr(), row, n, seqs, st["start"].data_ptr(),
                       st["len"].data_ptr(), stream=sp)
        dev.kv4_keep(cache, n, seqs, st["start"].data_ptr(), st["len"].data_ptr(), st["path"].data_ptr(),
                     st["count"].data_ptr(), sp)
        dev.kv4_read(cache, ty, st["kept"], seqs, st["kept_start"].data_ptr(), st["new_len"].data_ptr(),
                     st["k_out"].data_ptr(), row, st["v_out"].data_ptr(), row, sp)
        return [st["k_out"], st["v_out"]]
    row = c["heads"] * dim
    work = _kept(st, "work", lambda: _bytes(
        dev.kv4_tree_attention_work_bytes(cache, c["heads"], n, seqs, st["max_rows"])))
    dev.kv4_tree_attention(cache, ty, st["q"].data_ptr(), row, c["heads"], n, seqs, st["start"].data_ptr(),
                           st["max_rows"], st["len"].data_ptr(), st["mask"].data_ptr(), _words(c),
                           1.0 / math.sqrt(dim), st["out"].data_ptr(), row, work.data_ptr(), sp,
                           window=c["window"], lse=st["lse"].data_ptr())
    return [st["out"], st["lse"]]


def run(st):
    return _own_run(st) if own else _plain_run(st)


# ---- what a pass cannot do without -----------------------------------------

def work(case):
    c = case
    size = 4 if c["type"] == "f32" else 2
    if c["path"] in ("w8", "gated"):
        both = 1 if c["path"] == "w8" else 2
        return {"bytes": size * c["tokens"] * (c["in"] + c["out"]) + both * c["out"] * (c["in"] + 4),
                "flops": 2 * both * c["tokens"] * c["in"] * c["out"]}
    n = sum(_rows(c))
    if c["path"] == "accept":
        return {"bytes": size * n * c["vocab"] + 12 * n + 16 * c["seqs"], "flops": n * c["vocab"]}
    token = c["kv"] * c["dim"]  # a token's keys, or its values; 5 bits each in the cache
    if c["path"] == "keep":
        # All written; those kept moved (read and written, 5 bits each) and read back.
        kept = sum(_kept_rows(c))
        return {"bytes": int(token * (n * (2 * size + 2 * 5 / 8) + kept * (2 * size + 6 * 5 / 8))),
                "flops": n * token * 9}
    lens = _lens(c)
    seen = [min(m, c["window"] + r) if c["window"] else m for m, r in zip(lens, _rows(c))]
    return {"bytes": int(2 * sum(seen) * token * 5 / 8) + n * c["heads"] * (2 * c["dim"] * size + 4),
            "flops": 4 * c["dim"] * c["heads"] * sum(m * r for m, r in zip(seen, _rows(c)))}


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


def _exact_tokens(x):
    """(f64 scales, f64 codes) of tokens, a scale being the f32 next to max |x| / 127."""
    x = x.double()
    s = (x.abs().max(1).values / 127).float().double()
    below = torch.floor(x.abs() / s[:, None])  # the code or one less
    rest = x.abs() - below * s[:, None]
    up = (2 * rest > s[:, None]) | ((2 * rest == s[:, None]) & (below % 2 == 1))
    return s, torch.sign(x) * (below + up)


def exact(case, seed):
    if case["path"] == "accept":
        return None  # whole numbers, which have to be equal
    st = prepare(case, seed)
    c = case
    if c["path"] in ("w8", "gated"):
        s, q = _exact_tokens(st["x"])
        outs = []
        for name in (("w",) if c["path"] == "w8" else ("gate", "up")):
            y = torch.empty(c["tokens"], c["out"], dtype=torch.float64, device="cuda")
            for at in range(0, c["out"], 4096):
                w = st[name][at:at + 4096].double() * st[name + "_scale"][at:at + 4096].double()[:, None]
                y[:, at:at + 4096] = torch.mm(q * s[:, None], w.t().contiguous())
            outs.append(y)
        if c["path"] == "w8":
            return outs[0]
        g = outs[0]
        inner = math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)
        # gelu's 0.5 (1 + tanh t) is the logistic function of 2 t.
        return g * torch.sigmoid(g if c["act"] == "silu" else 2 * inner) * outs[1]
    kv, dim = c["kv"], c["dim"]
    start, parent = st["start"].tolist(), st["parent"].tolist()
    if c["path"] == "keep":
        path, count = st["path"].tolist(), st["count"].tolist()
        at = [start[b] + path[start[b] + i] for b in range(c["seqs"]) for i in range(count[b])]
        return [_exact_quantised(st[x].float()[at]) for x in ("k", "v")]
    outs, lses = [], []
    for b, (m, r) in enumerate(zip(st["lens"], st["rows"])):
        k, v = (_exact_cache(st, b, kind)[:, :m] for kind in ("k", "v"))
        see = torch.zeros(r, m, dtype=torch.bool)
        for i in range(r):
            on = [i]
            while parent[start[b] + on[-1]] >= 0:
                on.append(parent[start[b] + on[-1]])
            low = max(0, m - r - (c["window"] - len(on))) if c["window"] else 0
            see[i, low:m - r] = True
            see[i, [m - r + j for j in on]] = True
        see = see.cuda()
        q = st["q"][start[b]:start[b + 1]].double().view(r, kv, -1, dim)
        o, ls = [], []
        for h in range(kv):
            s = (q[:, h].reshape(-1, dim) @ k[h].t().contiguous() / math.sqrt(dim)).view(r, -1, m)
            s = s.masked_fill(~see[:, None], -math.inf)
            ls.append(torch.logsumexp(s, 2))
            o.append((torch.exp(s - ls[-1][..., None]).view(-1, m) @ v[h]).view(r, -1, dim))
        outs.append(torch.stack(o, 1).flatten(1, 2))
        lses.append(torch.stack(ls, 1).flatten(1, 2))
    return [torch.cat(outs), torch.cat(lses)]
