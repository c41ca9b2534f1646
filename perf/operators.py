"""Measured cases of the 4-bit KV cache's operators: block tables and slot maps
built from request lengths, K and V rows stored in 4 bits and read back, and
attention over the cache.

A page pool is uint8 [pages, kv_heads, page_bytes]. A page holds page_size
tokens in blocks of 16; a block of one head is, in this order:
  K codes   [16 tokens][D / 2 bytes]
  V codes   [16 tokens][D / 2 bytes]
  K params  [16 tokens][D / g] pairs (scale, zero) of fp16
  V params  [16 tokens][D / g] pairs (scale, zero) of fp16
A channel's value is code * scale + zero. Nibbles go low first. Nibble n of a
K row is channel 32 * w + 8 * t + i, where n counts (t, w, i) over
[4][D / 32][8]; nibble n of a V row is channel 8 * s + r, where n counts
(r, s) over [8][D / 8].
"""
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
F16_MAX = 65504.0


def listed():
    return [
        # the bookkeeping of one decode step of a small server: 17 requests, one token each
        {"name": "extend_step", "op": "extend", "batch": 17, "page": 16, "ctx": 900, "new_lo": 1, "new_hi": 1},
        # many prompts of mixed lengths admitted at once
        {"name": "extend_prompts", "op": "extend", "batch": 512, "page": 64, "ctx": 2048, "new_lo": 0, "new_hi": 255},
        # a few finished requests of a small batch give their pages back
        {"name": "release_step", "op": "release", "batch": 17, "page": 16, "ctx": 900},
        # half of a large batch of long requests ends
        {"name": "release_large", "op": "release", "batch": 512, "page": 16, "ctx": 8192},
        # one layer's new K and V rows of a 16-request decode step
        {"name": "append_step", "op": "append", "tokens": 16, "kv_heads": 8, "dim": 128, "g": 64, "page": 64, "dtype": "fp16"},
        # one layer's K and V rows of prompts, at a length that fills no page evenly
        {"name": "append_prompt", "op": "append", "tokens": 8191, "kv_heads": 8, "dim": 128, "g": 64, "page": 64, "dtype": "bf16"},
        # the 7B decoder's attention step: 32 heads, a 2048-token cache and the new token
        {"name": "attend_7b_step", "op": "attend", "batch": 1, "kv_heads": 32, "share": 1, "dim": 128, "g": 128, "page": 64,
         "ctx_lo": 2049, "ctx_hi": 2049, "new_lo": 1, "new_hi": 1, "dtype": "fp16"},
        # a small model's heads, short ragged requests, small pages: latency counts
        {"name": "attend_small_ragged", "op": "attend", "batch": 24, "kv_heads": 2, "share": 7, "dim": 64, "g": 32, "page": 16,
         "ctx_lo": 0, "ctx_hi": 999, "new_lo": 1, "new_hi": 1, "dtype": "bf16"},
        # a decode step of a busy server: ragged contexts, heads shared by four
        {"name": "attend_batch", "op": "attend", "batch": 32, "kv_heads": 8, "share": 4, "dim": 128, "g": 64, "page": 64,
         "ctx_lo": 4000, "ctx_hi": 8192, "new_lo": 1, "new_hi": 1, "dtype": "fp16"},
        # one long document: the keys of few rows split over the whole GPU
        {"name": "attend_long", "op": "attend", "batch": 1, "kv_heads": 8, "share": 8, "dim": 128, "g": 64, "page": 64,
         "ctx_lo": 131071, "ctx_hi": 131071, "new_lo": 1, "new_hi": 1, "dtype": "bf16"},
        # a few guessed tokens of each request checked in one pass
        {"name": "attend_verify", "op": "attend", "batch": 16, "kv_heads": 8, "share": 4, "dim": 128, "g": 32, "page": 32,
         "ctx_lo": 1500, "ctx_hi": 4001, "new_lo": 3, "new_hi": 6, "dtype": "fp16"},
        # prompt chunks behind contexts that are in the cache already
        {"name": "attend_prompt", "op": "attend", "batch": 4, "kv_heads": 8, "share": 4, "dim": 128, "g": 64, "page": 64,
         "ctx_lo": 2500, "ctx_hi": 4096, "new_lo": 500, "new_hi": 1024, "dtype": "fp16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["extend", "release", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if op in ("extend", "release"):
        c = {"op": op, "batch": _log_int(rng, 1, 512), "page": page, "ctx": _log_int(rng, 16, 8192 if op == "release" else 2048)}
        if op == "extend":
            hi = _log_int(rng, 1, 255)
            c |= {"new_lo": rng.choice([0, 1, hi]), "new_hi": hi}
        return c
    dim = rng.choice([64, 128])
    g = rng.choice([x for x in (32, 64, 128) if x <= dim])
    dtype = rng.choice(["fp16", "bf16"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    if op == "append":
        return {"op": op, "tokens": _log_int(rng, 1, 8191), "kv_heads": kv_heads, "dim": dim, "g": g, "page": page, "dtype": dtype}
    share = rng.choice([1, 2, 3, 4, 7, 8])
    batch = _log_int(rng, 1, 32)
    most = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 16, 1024)])
    # keys of all requests and heads, and query-key pairs, stay below those of the largest listed cases
    room = min(131071 * 8 // (batch * kv_heads), 4 * 1024 * 4096 * 32 // (batch * most * kv_heads * share))
    ctx = max(most, _log_int(rng, 1, max(1, min(131071, room))))
    return {"op": op, "batch": batch, "kv_heads": kv_heads, "share": share, "dim": dim, "g": g, "page": page,
            "ctx_lo": max(most, rng.choice([ctx, ctx // 2, ctx // 9])), "ctx_hi": ctx, "new_lo": rng.randint(1, most), "new_hi": most, "dtype": dtype}


# -- the cache's layout in elementary operations ---------------------------------

def _block_bytes(dim, g):
    return 16 * dim + 16 * 8 * (dim // g)


def _quantise(x, g):
    """fp32 rows [..., D] -> codes uint8 [..., D], params fp16 [..., D / g, 2] (scale, zero)."""
    x = x.float().clamp(-F16_MAX, F16_MAX)
    xg = x.reshape(*x.shape[:-1], -1, g)
    lo, hi = xg.amin(-1), xg.amax(-1)
    zero = lo.to(torch.float16)
    scale = ((hi - lo) / torch.full_like(lo, 15.0)).to(torch.float16)
    s, z = scale.float().unsqueeze(-1), zero.float().unsqueeze(-1)
    code = torch.round((xg - z) / torch.where(s == 0, torch.ones_like(s), s)).clamp(0, 15)
    code = torch.where(s == 0, torch.zeros_like(code), code).to(torch.uint8)
    return code.reshape(x.shape), torch.stack((scale, zero), dim=-1)


def _values(code, par, g):
    v = code.float().reshape(*code.shape[:-1], -1, g) * par[..., 0:1].float() + par[..., 1:2].float()
    return v.reshape(code.shape)


def _order(code, is_v):
    """Channel order -> nibble order."""
    lead, dim = code.shape[:-1], code.shape[-1]
    c = code.reshape(*lead, dim // 8, 8) if is_v else code.reshape(*lead, dim // 32, 4, 8)
    return (c.transpose(-1, -2) if is_v else c.transpose(-2, -3)).reshape(*lead, dim)


def _unorder(code, is_v):
    """Nibble order -> channel order."""
    lead, dim = code.shape[:-1], code.shape[-1]
    c = code.reshape(*lead, 8, dim // 8) if is_v else code.reshape(*lead, 4, dim // 32, 8)
    return (c.transpose(-1, -2) if is_v else c.transpose(-2, -3)).reshape(*lead, dim)


def _pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _unpack(b):
    return torch.stack((b & 15, b >> 4), dim=-1).flatten(-2)


def _views(pool, dim, g):
    """The four parts of a pool: K codes, V codes [N, H, blocks, 16, D / 2] and params [N, H, blocks, 16, D / g, 2]."""
    n, h, nb = pool.shape[0], pool.shape[1], pool.shape[2] // _block_bytes(dim, g)
    blk = pool.view(n, h, nb, _block_bytes(dim, g))
    c, p = 16 * dim // 2, 16 * 4 * (dim // g)
    kc = blk[..., :c].unflatten(-1, (16, dim // 2))
    vc = blk[..., c:2 * c].unflatten(-1, (16, dim // 2))
    kp = blk[..., 2 * c:2 * c + p].view(torch.float16).unflatten(-1, (16, dim // g, 2))
    vp = blk[..., 2 * c + p:].view(torch.float16).unflatten(-1, (16, dim // g, 2))
    return kc, vc, kp, vp


def _store(pool, k, v, slots, dim, g):
    """Rows k, v [T, H, D] at slots [T] (-1: none), in place."""
    keep = slots >= 0
    s = slots[keep].long()
    page = pool.shape[2] // _block_bytes(dim, g) * 16
    n, b, t = s // page, (s % page) // 16, s % 16
    kc, vc, kp, vp = _views(pool, dim, g)
    for x, codes, params, is_v in ((k, kc, kp, False), (v, vc, vp, True)):
        code, par = _quantise(x[keep], g)
        codes[n, :, b, t] = _pack(_order(code, is_v))
        params[n, :, b, t] = par


# -- inputs ---------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randint(gen, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=gen, device="cuda", dtype=torch.int32)


def _rows(gen, n, heads, dim, dtype, keys):
    """K or V rows: normal, keys with the few strong channels that a model's keys have."""
    x = torch.randn(n, heads, dim, generator=gen, device="cuda")
    if keys:
        off = torch.randn(heads, dim, generator=gen, device="cuda")
        x = x + torch.where(off.abs() > 2, 3 * off, torch.zeros_like(off))
    return x.to(dtype)


def prepare(case, seed):
    gen = _gen(seed)
    op, page = case["op"], case["page"]
    if op in ("extend", "release"):
        # a server in mid-run: every request has its pages, the other pages lie on the free stack, lowest last
        batch = case["batch"]
        lens = _randint(gen, 0, case["ctx"], batch)
        new = _randint(gen, case.get("new_lo", 0), case.get("new_hi", 0), batch)
        width = -(-(case["ctx"] + case.get("new_hi", 0)) // page)
        total = batch * width
        ids = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
        held = (lens + page - 1) // page
        col = torch.arange(width, device="cuda", dtype=torch.int32)
        first = torch.cumsum(held, 0, dtype=torch.int32) - held
        table = torch.where(col < held[:, None], ids[(first[:, None] + col).clamp(max=total - 1).long()], torch.full_like(ids[:1], -1))
        used = held.sum(dtype=torch.int32)
        at = torch.arange(total, device="cuda", dtype=torch.int32)
        free = torch.where(at < total - used, ids[(at + used).clamp(max=total - 1).long()], torch.full_like(at, -1))
        return {"op": op, "page": page, "lens": lens, "new": new, "table": table.contiguous(), "free": free,
                "count": (total - used).reshape(1), "max_tokens": batch * case.get("new_hi", 0),
                "done": (torch.rand(batch, generator=gen, device="cuda") < 0.5)}
    dim, g, heads, dtype = case["dim"], case["g"], case["kv_heads"], DTYPES[case["dtype"]]
    page_bytes = page // 16 * _block_bytes(dim, g)
    if op == "append":
        # the rows of a step, at slots spread over the pool as the tables give them
        n = case["tokens"]
        pages = -(-n // page) + 8
        pool = torch.full((pages, heads, page_bytes), 255, dtype=torch.uint8, device="cuda")
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:n].to(torch.int32)
        if n > page:  # a prompt's tokens lie one after another in its pages
            order = torch.randperm(pages, generator=gen, device="cuda")[: -(-n // page)]
            slots = (order[:, None] * page + torch.arange(page, device="cuda")).flatten()[:n].to(torch.int32)
        return {"op": op, "k": _rows(gen, n, heads, dim, dtype, True), "v": _rows(gen, n, heads, dim, dtype, False),
                "pool": pool, "slots": slots, "dim": dim, "g": g, "dtype": dtype}
    batch = case["batch"]
    lens = _randint(gen, case["ctx_lo"], case["ctx_hi"], batch)
    lens[batch // 2] = case["ctx_hi"]
    # how many new tokens each request has is the case's: the outputs' shape goes by it
    spread = case["new_hi"] - case["new_lo"] + 1
    new = (case["new_lo"] + torch.arange(batch, device="cuda", dtype=torch.int32) * 7919 % spread).to(torch.int32)
    width = -(-case["ctx_hi"] // page)
    held = (lens + page - 1) // page
    pages = int(held.sum()) + 4
    # what is not written yet holds 255 in every byte, which is NaN as a scale or a zero
    pool = torch.full((pages, heads, page_bytes), 255, dtype=torch.uint8, device="cuda")
    ids = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, (n, m) in enumerate(zip(lens.tolist(), held.tolist())):
        table[b, :m] = ids[at:at + m]
        at += m
        pos = torch.arange(n, device="cuda")
        slots = table[b, pos // page].long() * page + pos % page
        for c in range(0, n, 16384):
            s = slots[c:c + 16384]
            _store(pool, _rows(gen, len(s), heads, dim, dtype, True), _rows(gen, len(s), heads, dim, dtype, False), s, dim, g)
    starts = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    starts[1:] = torch.cumsum(new, 0, dtype=torch.int32)
    q = torch.randn(int(starts[-1]), heads * case["share"], dim, generator=gen, device="cuda").to(dtype)
    # a step of one token each has no starts
    one = case["new_hi"] == 1
    return {"op": op, "q": q, "pool": pool, "table": table, "lens": lens, "starts": None if one else starts,
            "max_new": case["new_hi"], "g": g, "dtype": dtype}


# -- the operators --------------------------------------------------------------

def run(state):
    op = state["op"]
    if own:
        import ecq_b200 as ecq

        if op == "extend":
            step = ecq.kv4_extend(state["lens"], state["new"], state["table"], state["free"], state["count"], state["page"],
                                  state["max_tokens"])
            return [step.seq_lens, step.q_starts, step.slots, step.positions, step.free_count, state["table"]]
        if op == "release":
            lens, count = ecq.kv4_release(state["done"], state["lens"], state["table"], state["free"], state["count"], state["page"])
            return [lens, count, state["free"]]
        if op == "append":
            ecq.kv4_append(state["k"], state["v"], state["pool"], state["slots"], group_size=state["g"])
            return list(ecq.kv4_gather(state["pool"], state["slots"], state["dim"], group_size=state["g"], dtype=state["dtype"]))
        return ecq.kv4_attention(state["q"], state["pool"], state["table"], state["lens"], state["starts"], state["max_new"],
                                 group_size=state["g"])
    if op == "extend":
        return _extend(state)
    if op == "release":
        return _release(state)
    if op == "append":
        return _append(state)
    return _attend(state)


def _extend(st):
    lens, new, page, table, free = st["lens"], st["new"], st["page"], st["table"], st["free"]
    after = lens + new
    held, need = (lens + page - 1) // page, (after + page - 1) // page
    take = need - held
    first = torch.cumsum(take, 0, dtype=torch.int32) - take
    col = torch.arange(table.shape[1], device=table.device, dtype=torch.int32)
    fresh = (col >= held[:, None]) & (col < need[:, None])
    place = st["count"] - 1 - (first[:, None] + col - held[:, None])
    table.copy_(torch.where(fresh, free[place.clamp(0, free.numel() - 1).long()], table))
    starts = torch.zeros(lens.numel() + 1, dtype=torch.int32, device=lens.device)
    starts[1:] = torch.cumsum(new, 0, dtype=torch.int32)
    i = torch.arange(st["max_tokens"], device=lens.device, dtype=torch.int32)
    b = torch.searchsorted(starts[1:], i, right=True).clamp(max=lens.numel() - 1)
    valid = i < starts[-1]
    pos = torch.where(valid, lens[b] + i - starts[b], torch.zeros_like(i))
    slots = table[b, (pos // page).clamp(max=table.shape[1] - 1).long()] * page + pos % page
    none = torch.full_like(i, -1)
    return [after, starts, torch.where(valid, slots, none), torch.where(valid, pos, none), st["count"] - take.sum(dtype=torch.int32), table]


def _release(st):
    lens, page, table, free, count = st["lens"], st["page"], st["table"], st["free"], st["count"]
    back = torch.where(st["done"], (lens + page - 1) // page, torch.zeros_like(lens))
    first = torch.cumsum(back, 0, dtype=torch.int32) - back
    col = torch.arange(table.shape[1], device=table.device, dtype=torch.int32)
    given = col < back[:, None]
    free[(count + first[:, None] + col)[given].long()] = table[given]
    return [torch.where(st["done"], torch.zeros_like(lens), lens), count + back.sum(dtype=torch.int32), free]


def _append(st):
    dim, g, pool, dtype = st["dim"], st["g"], st["pool"], st["dtype"]
    _store(pool, st["k"], st["v"], st["slots"], dim, g)
    s = st["slots"].long()
    page = pool.shape[2] // _block_bytes(dim, g) * 16
    n, b, t = s // page, (s % page) // 16, s % 16
    kc, vc, kp, vp = _views(pool, dim, g)
    return [_values(_unorder(_unpack(kc[n, :, b, t]), False), kp[n, :, b, t], g).to(dtype),
            _values(_unorder(_unpack(vc[n, :, b, t]), True), vp[n, :, b, t], g).to(dtype)]


def _attend(st):
    q, pool, g, lens, table = st["q"], st["pool"], st["g"], st["lens"], st["table"]
    dim, heads = q.shape[2], pool.shape[1]
    share, batch = q.shape[1] // heads, lens.numel()
    idx = table.clamp(min=0).long()
    kc, vc, kp, vp = (x[idx].transpose(1, 2) for x in _views(pool, dim, g))  # [B, H, pages, blocks, 16, ...]
    k = _values(_unorder(_unpack(kc), False), kp, g).flatten(2, 4)          # [B, H, L, D]
    v = _values(_unorder(_unpack(vc), True), vp, g).flatten(2, 4)
    j = torch.arange(k.shape[2], device=q.device)
    inside = j < lens[:, None]                                               # [B, L]
    v = torch.where(inside[:, None, :, None], v, torch.zeros_like(v))
    starts = st["starts"] if st["starts"] is not None else torch.arange(batch + 1, device=q.device, dtype=torch.int32)
    new = starts[1:] - starts[:-1]
    i = torch.arange(st["max_new"], device=q.device, dtype=torch.int32)
    at = (starts[:-1, None] + i).clamp(max=max(0, q.shape[0] - 1)).long()    # [B, n]: padded to the longest
    qp = q[at].float().unflatten(2, (heads, share)).permute(0, 2, 3, 1, 4)   # [B, H, share, n, D]
    s = torch.matmul(qp.flatten(2, 3), k.transpose(-1, -2)).unflatten(2, (share, st["max_new"])) * dim ** -0.5
    seen = j <= (lens[:, None] - new[:, None] + i)[..., None]                # [B, n, L]
    seen = (seen & inside[:, None, :])[:, None, None]
    s = torch.where(seen, s, torch.full_like(s, float("-inf")))
    m = s.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(s - m), torch.zeros_like(s))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.flatten(2, 3), v).unflatten(2, (share, st["max_new"])) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)                               # [B, n, heads, D]
    t = torch.arange(q.shape[0], device=q.device, dtype=torch.int32)
    b = torch.searchsorted(starts[1:], t, right=True)
    return o[b, (t - starts[b]).long()].to(st["dtype"])


# -- the definition in 64 bits, request by request -------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    op = st["op"]
    if op in ("extend", "release"):
        return None  # whole numbers
    g = st["g"]
    if op == "append":
        out = []
        for x in (st["k"], st["v"]):
            y = x.double().view(*x.shape[:2], -1, g)
            lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
            zero, scale = lo.half().double(), ((hi - lo) / 15).half().double()
            code = ((y - zero) / scale.clamp(min=2.0 ** -24)).round().clamp(0, 15)
            out.append((code * scale + zero).view(x.shape))
        return out
    q, pool, table, page = st["q"].double(), st["pool"], st["table"], case["page"]
    dim, heads, share = case["dim"], case["kv_heads"], case["share"]
    d = torch.arange(dim, device=q.device)
    nib = {False: ((d % 32) // 8) * (dim // 4) + (d // 32) * 8 + d % 8, True: (d % 8) * (dim // 8) + d // 8}
    block, out = _block_bytes(dim, g), torch.zeros_like(q)
    starts = list(range(case["batch"] + 1)) if st["starts"] is None else st["starts"].tolist()
    for b, n in enumerate(st["lens"].tolist()):
        lo, hi = starts[b], starts[b + 1]
        if n == 0 or hi == lo:
            continue
        pos = torch.arange(n, device=q.device)
        blk = pool[table[b, :-(-n // page)].long()].view(-1, heads, page // 16, block)
        kv = []
        for is_v in (False, True):
            code = blk[..., 8 * dim * is_v:][..., :8 * dim].unflatten(-1, (16, dim // 2))[..., nib[is_v] // 2]
            code = code >> ((nib[is_v] % 2) * 4).to(torch.uint8) & 15
            par = blk[..., 16 * dim:].contiguous().view(torch.float16).unflatten(-1, (2, 16, dim // g, 2))[..., int(is_v), :, :, :]
            x = code.double() * par[..., d // g, 0] + par[..., d // g, 1]       # [pages, H, blocks, 16, D]
            kv.append(x.transpose(0, 1).reshape(heads, -1, dim)[:, :n])
        where = n - (hi - lo) + torch.arange(hi - lo, device=q.device)
        for h in range(heads):
            x = q[lo:hi, h * share:(h + 1) * share].transpose(0, 1)
            s = x @ kv[0][h].t() / dim ** 0.5
            s = s.masked_fill(pos > where[:, None], -float("inf"))
            out[lo:hi, h * share:(h + 1) * share] = (torch.softmax(s, -1) @ kv[1][h]).transpose(0, 1)
    return out


def _mean(lo, hi):
    return (lo + hi) / 2


def work(case):
    op = case["op"]
    if op in ("extend", "release"):
        b, new = case["batch"], _mean(case.get("new_lo", 0), case.get("new_hi", 0))
        pages = b * (new if op == "extend" else case["ctx"] / 4) / case["page"]
        # lengths in and out, counts, starts; a table entry and a stack entry for each page; slot and position of each token
        return {"bytes": 4 * (4 * b + 3) + 8 * pages + (8 * b * case.get("new_hi", 0) if op == "extend" else 0), "flops": 8 * b + 4 * b * new}
    row = case["dim"] + 8 * (case["dim"] // case["g"])  # bytes of K and V of a token and head in the cache
    if op == "append":
        n = case["tokens"] * case["kv_heads"]
        # rows in, packed out; packed in, rows out
        return {"bytes": n * (2 * 4 * case["dim"] + 2 * row) + 8 * case["tokens"], "flops": n * case["dim"] * 2 * 10}
    b, heads = case["batch"], case["kv_heads"] * case["share"]
    keys, new = _mean(case["ctx_lo"], case["ctx_hi"]), _mean(case["new_lo"], case["new_hi"])
    pairs = b * new * max(1.0, keys - (new - 1) / 2)
    return {"bytes": b * (keys * case["kv_heads"] * row + 4 * keys / case["page"] + 8) + 4 * b * new * heads * case["dim"],
            "flops": 4 * case["dim"] * heads * pairs}
