"""What is measured of the 4-bit KV cache: writing it and the two forms of attention that read it.

``append``   RMS norm of every query and key head, the position rotation, and the write of keys and values into
             the paged 4-bit cache, for a batch of token rows.
``decode``   one new token per sequence: norm and rotation of its heads, the write of its row, and attention over
             the sequence's cached rows.
``prompt``   causal attention of the consecutive rows of a prompt chunk over the sequence's cached rows.

A page of the cache holds 16 tokens of one kv head: 16 rows of ``head_dim / 2`` bytes of codes, in the order in which
the matrix instruction takes them, and behind them for every token a bf16 scale and a bf16 minimum.  A value is
``code * scale + minimum`` with a code of 0 .. 15, one scale and one minimum to a (token, kv head) row.
The caches are returned as the bytes they hold: whole pages, rows that were not written included."""
import math

import torch

own = False

PAGE = 16
LIMIT = 32768.0            # keys and values are held within +-LIMIT
DEV = "cuda"


def listed():
    return [
        # -- append: one row of a decode step that runs as a token batch (partial rotation, adjacent heads as in the 32-head, 80-wide shape)
        dict(name="append-1row-80", op="append", rows=1, heads=32, kv_heads=32, head_dim=80, norm=False, rope_dim=32, rope_type=2, idle=0),
        # a ragged batch of rows of a small model, some of them idle
        dict(name="append-333-64", op="append", rows=333, heads=14, kv_heads=2, head_dim=64, norm=False, rope_dim=64, rope_type=2, idle=5),
        # a default prompt chunk of a model that normalises queries and keys
        dict(name="append-512-128", op="append", rows=512, heads=32, kv_heads=8, head_dim=128, norm=True, rope_dim=128, rope_type=2, idle=0),
        # a long prompt in one pass
        dict(name="append-8192-128", op="append", rows=8192, heads=32, kv_heads=8, head_dim=128, norm=True, rope_dim=128, rope_type=0, idle=0),
        # -- decode: the batch-1 step of the 32-head, 80-wide shape
        dict(name="decode-1x640-80", op="decode", batch=1, heads=32, kv_heads=32, head_dim=80, ctx=640, ragged=False, window=0, norm=False, rope_dim=32, rope_type=2),
        # one sequence with a very long context
        dict(name="decode-1x131072-128", op="decode", batch=1, heads=32, kv_heads=8, head_dim=128, ctx=131072, ragged=False, window=0, norm=True, rope_dim=128, rope_type=2),
        # an odd batch of unequal lengths with a sliding window, seven query heads to a kv head
        dict(name="decode-37x4000-64", op="decode", batch=37, heads=14, kv_heads=2, head_dim=64, ctx=4000, ragged=True, window=1000, norm=False, rope_dim=64, rope_type=2),
        # a full serving batch
        dict(name="decode-64x2048-128", op="decode", batch=64, heads=32, kv_heads=8, head_dim=128, ctx=2048, ragged=False, window=0, norm=False, rope_dim=128, rope_type=0),
        # the largest: a serving batch of long, unequal sequences
        dict(name="decode-96x8192-128", op="decode", batch=96, heads=32, kv_heads=8, head_dim=128, ctx=8192, ragged=True, window=0, norm=True, rope_dim=128, rope_type=2),
        # -- prompt: a short continuation at an odd position
        dict(name="prompt-77at1337-64", op="prompt", rows=77, pos0=1337, heads=14, kv_heads=2, head_dim=64, window=0),
        # a default chunk in the middle of a prompt
        dict(name="prompt-512at1536-128", op="prompt", rows=512, pos0=1536, heads=32, kv_heads=8, head_dim=128, window=0),
        # a large chunk behind a long context
        dict(name="prompt-2048at6144-128", op="prompt", rows=2048, pos0=6144, heads=32, kv_heads=8, head_dim=128, window=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "prompt"])
    d = rng.choice([64, 80, 96, 128])
    kvh = rng.choice([1, 2, 4, 8, 8, 16, 32])
    g = rng.choice([1, 2, 3, 4, 5, 7, 8, 12]) if kvh <= 4 else rng.choice([1, 2, 4, 4, 5]) if kvh <= 16 else 1
    h = kvh * g
    rope_dim = rng.choice([d, d, d // 2, 32])
    rope_type = rng.choice([0, 2])
    norm = rng.random() < 0.5
    if op == "append":
        rows = _log(rng, 1, min(8192, 50_000_000 // ((h + 2 * kvh) * d)))
        return dict(op=op, rows=rows, heads=h, kv_heads=kvh, head_dim=d, norm=norm, rope_dim=rope_dim, rope_type=rope_type, idle=rng.choice([0, 0, rows // 9]))
    if op == "decode":
        batch = _log(rng, 1, 128)
        most = min(131072, 64 * 8192 * 8 * 128 // (batch * kvh * d))
        ctx = _log(rng, 1, max(2, most))
        return dict(op=op, batch=batch, heads=h, kv_heads=kvh, head_dim=d, ctx=ctx, ragged=rng.random() < 0.5, window=rng.choice([0, 0, 0, 1 + ctx // 3]),
                    norm=norm, rope_dim=rope_dim, rope_type=rope_type)
    rows = _log(rng, 1, 2048)
    most = 2048 * 8192 * 32 * 128 // (rows * h * d) - rows
    pos0 = rng.choice([0, _log(rng, 1, min(32768, most)) if most > 1 else 0])
    return dict(op=op, rows=rows, pos0=pos0, heads=h, kv_heads=kvh, head_dim=d, window=rng.choice([0, 0, 1 + (pos0 + rows) // 3]))


# ---- the inputs ---------------------------------------------------------------------------------------------------------
def _row_bytes(d):
    return d // 2 + 4


def _cache(gen, pages, kvh, d, spread):
    """Codes of a normal distribution around the middle of the range, a scale and a minimum to each row."""
    n = pages * kvh * PAGE
    lo = (torch.randn(n, d // 2, generator=gen, device=DEV, dtype=torch.float16) * 3.0 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    hi = (torch.randn(n, d // 2, generator=gen, device=DEV, dtype=torch.float16) * 3.0 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    codes = (hi << 4 | lo).view(pages, kvh, PAGE * d // 2)
    scale = (spread * (0.75 + 0.5 * torch.rand(n, generator=gen, device=DEV))).to(torch.bfloat16)
    low = (scale.float() * (-7.5 + torch.randn(n, generator=gen, device=DEV))).to(torch.bfloat16)
    meta = torch.stack([scale, low], -1).view(torch.uint8).view(pages, kvh, PAGE * 4)
    return torch.cat([codes, meta], -1).view(pages, kvh, PAGE, _row_bytes(d)).contiguous()


def _rope_table(positions, rope_dim, theta=10000.0):
    i = torch.arange(rope_dim // 2, dtype=torch.float64, device=DEV)
    ang = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * torch.pow(torch.tensor(theta, dtype=torch.float64, device=DEV), -2.0 * i / rope_dim)
    return torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()


def _lengths(c):
    if not c["ragged"]:
        return [c["ctx"]] * c["batch"]
    return [max(1, c["ctx"] - (b * 7919) % max(1, c["ctx"] * 2 // 3)) for b in range(c["batch"])]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    h, kvh, d = c["heads"], c["kv_heads"], c["head_dim"]
    rnd = lambda *s: torch.randn(*s, generator=gen, device=DEV)                                     # noqa: E731
    s = dict(c)
    if c["op"] == "append":
        n = c["rows"]
        np_seq = 24                                                                                  # rows of several sequences, 24 pages each
        pages = -(-n // (np_seq * PAGE)) * np_seq + 3
        perm = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
        at = torch.arange(n, device=DEV)
        s["positions"] = (at % (np_seq * PAGE)).to(torch.int32)
        s["page_rows"] = perm[(at // PAGE)].contiguous()
        if c["idle"]:
            s["positions"][torch.randperm(n, generator=gen, device=DEV)[: c["idle"]]] = -1
        s["q_out"] = torch.zeros(n, h * d, device=DEV)
        table_len = np_seq * PAGE
    elif c["op"] == "decode":
        n, lens = c["batch"], _lengths(c)
        per = -(-max(lens) // PAGE)
        pages = n * per + 3
        s["page_table"] = torch.randperm(pages, generator=gen, device=DEV)[: n * per].to(torch.int32).view(n, per).contiguous()
        s["positions"] = torch.tensor([v - 1 for v in lens], dtype=torch.int32, device=DEV)
        s["out"] = torch.zeros(n, h * d, device=DEV)
        table_len = max(lens)
    else:
        n, total = c["rows"], c["pos0"] + c["rows"]
        per = -(-total // PAGE)
        pages = per + 3
        s["page_table"] = torch.randperm(pages, generator=gen, device=DEV)[:per].to(torch.int32).contiguous()
        s["out"] = torch.zeros(n, h * d, device=DEV, dtype=torch.bfloat16)
    s["qkv"] = rnd(n, (h + 2 * kvh) * d)
    s["k_cache"], s["v_cache"] = _cache(gen, pages, kvh, d, 0.33), _cache(gen, pages, kvh, d, 0.33)
    if c["op"] != "prompt":
        s["q_norm_w"] = 1 + 0.1 * rnd(d) if c["norm"] else None
        s["k_norm_w"] = 1 + 0.1 * rnd(d) if c["norm"] else None
        s["rope_table"] = _rope_table(table_len, c["rope_dim"])
    if own:                                                    # what a serving program sets up once: workspaces and the launch description
        from realizar_b200 import ops
        if c["op"] == "decode":
            s["scratch"] = ops.attn_decode_scratch(n, h, 1, d, DEV, kv_dtype="q4")
            s["plan"] = ops.build_attn_decode_params(s["qkv"], s["out"], s["k_cache"], s["v_cache"], s["positions"], s["page_table"], *s["scratch"],
                                                     h, kvh, d, 1, n, c["rope_dim"], c["rope_type"], 10000.0, 0, h * d, (h + kvh) * d,
                                                     s["q_norm_w"], s["k_norm_w"], 1e-6, window=c["window"], rope_table=s["rope_table"])
        elif c["op"] == "prompt":
            s["scratch"] = ops.attn_prefill_scratch(n, h, kvh, d, DEV)
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------------
def _offsets(d):
    """Byte of a page's code area that holds dims (2b, 2b+1) of token t, for keys and for values: [16, d / 2] each."""
    t, b = torch.arange(PAGE, device=DEV)[:, None], torch.arange(d // 2, device=DEV)[None, :]
    full = d // 32
    w = b // 4
    k = t * (d // 2) + torch.where(w < 4 * full, w % 4 * full + w // 4, w) * 4 + b % 4
    half, pair, odd, e = t // 8, t % 8 // 2, t % 2, b // 2
    v = (((half * 8 + e % 8) * 4 + pair) * full + e // 8) * 4 + odd * 2 + b % 2
    tail = 256 * full + ((b - 16 * full) * 4 + pair) * 4 + half * 2 + odd
    return k, torch.where(b < 16 * full, v, tail)


def _values(pages, offsets, d):
    """fp32 values of whole pages [..., 16, d / 2 + 4] -> [..., 16, d]."""
    flat = pages.flatten(-2)
    byte = flat[..., offsets]
    codes = torch.stack([byte & 15, byte >> 4], -1).flatten(-2).float()
    meta = flat[..., 8 * d:].contiguous().view(torch.bfloat16).unflatten(-1, (PAGE, 2)).float()
    return codes * meta[..., :1] + meta[..., 1:]


def _write(cache, rows, offsets, pages, slots, d):
    """Quantise fp32 rows [n, kv heads, d] and write them at (page, slot); rows with a page of -1 are left out."""
    keep = pages >= 0
    rows, pages, slots = rows[keep], pages[keep].long(), slots[keep].long()
    x = torch.where(torch.isnan(rows), torch.zeros_like(rows), rows).clamp(-LIMIT, LIMIT)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale, low = ((high - low) / torch.full_like(low, 15.0)).bfloat16(), low.bfloat16()             # (a divisor that is a plain number would be a product)
    code = ((x.double() - low.double()) / scale.double()).round().clamp(0, 15)                       # in 64 bits: values lie next to a border
    code = torch.where(scale.double() > 0, code, torch.zeros_like(code)).to(torch.uint8)
    byte = code[..., 0::2] | code[..., 1::2] << 4
    flat = cache.flatten(-2)
    head = torch.arange(cache.shape[1], device=DEV)[None, :, None]
    flat[pages[:, None, None], head, offsets[slots][:, None, :]] = byte
    meta = torch.cat([scale, low], -1).view(torch.uint8)
    flat[pages[:, None, None], head, (8 * d + 4 * slots[:, None] + torch.arange(4, device=DEV))[:, None, :]] = meta


def _norm_rope(x, w, positions, table, c):
    """RMS norm over the last axis and rotation of its first ``rope_dim`` values, in the type of ``x`` [n, heads, d]."""
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.to(x.dtype)
    r = c["rope_dim"]
    cs = table[positions.clamp(min=0).long()].to(x.dtype)[:, None]
    cos, sin = cs[..., 0], cs[..., 1]
    rot = x[..., :r]
    if c["rope_type"] == 2:
        a, b = rot[..., : r // 2], rot[..., r // 2:]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = rot[..., 0::2], rot[..., 1::2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _split(s):
    n, h, kvh, d = s["qkv"].shape[0], s["heads"], s["kv_heads"], s["head_dim"]
    q, k, v = s["qkv"].split([h * d, kvh * d, kvh * d], -1)
    return q.view(n, h, d), k.view(n, kvh, d), v.view(n, kvh, d)


def _softmax(x):
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_append(s):
    q, k, v = _split(s)
    d, pos = s["head_dim"], s["positions"]
    ok, ov = _offsets(d)
    live = pos >= 0
    turned = _norm_rope(q, s["q_norm_w"], pos, s["rope_table"], s).flatten(1)
    s["q_out"].copy_(torch.where(live[:, None], turned, s["q_out"]))
    pages = torch.where(live, s["page_rows"], torch.full_like(s["page_rows"], -1))
    key = _norm_rope(k.double(), s["k_norm_w"], pos, s["rope_table"], s).float()                     # in 64 bits: its codes lie next to a border
    _write(s["k_cache"], key, ok, pages, pos % PAGE, d)
    _write(s["v_cache"], v, ov, pages, pos % PAGE, d)
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_decode(s):
    q, k, v = _split(s)
    h, kvh, d, pos, pt = s["heads"], s["kv_heads"], s["head_dim"], s["positions"], s["page_table"]
    ok, ov = _offsets(d)
    n = q.shape[0]
    q = _norm_rope(q, s["q_norm_w"], pos, s["rope_table"], s)
    key = _norm_rope(k.double(), s["k_norm_w"], pos, s["rope_table"], s).float()
    page = pt.gather(1, (pos // PAGE).long()[:, None])[:, 0]
    _write(s["k_cache"], key, ok, page, pos % PAGE, d)
    _write(s["v_cache"], v, ov, page, pos % PAGE, d)
    keys = _values(s["k_cache"][pt.long()], ok, d).transpose(1, 2).flatten(2, 3)                     # [n, kv heads, positions, d]
    x = torch.matmul(q.view(n, kvh, h // kvh, d), keys.transpose(-1, -2)) * d ** -0.5
    del keys
    at = torch.arange(x.shape[-1], device=DEV)
    hidden = at > pos[:, None]
    if s["window"]:
        hidden = hidden | (at <= pos[:, None] - s["window"])
    x = _softmax(x.masked_fill(hidden[:, None, None], -math.inf))
    vals = _values(s["v_cache"][pt.long()], ov, d).transpose(1, 2).flatten(2, 3)
    s["out"].copy_(torch.matmul(x, vals).reshape(n, h * d))
    return {"out": s["out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_prompt(s):
    q, _, _ = _split(s)
    h, kvh, d, pt = s["heads"], s["kv_heads"], s["head_dim"], s["page_table"].long()
    ok, ov = _offsets(d)
    n = q.shape[0]
    keys = _values(s["k_cache"][pt], ok, d).transpose(0, 1).flatten(1, 2)                            # [kv heads, positions, d]
    x = torch.matmul(q.view(n, kvh, h // kvh, d).permute(1, 2, 0, 3), keys[:, None].transpose(-1, -2)) * d ** -0.5
    pos = s["pos0"] + torch.arange(n, device=DEV)
    at = torch.arange(x.shape[-1], device=DEV)
    hidden = at > pos[:, None]
    if s["window"]:
        hidden = hidden | (at <= pos[:, None] - s["window"])
    x = _softmax(x.masked_fill_(hidden, -math.inf))
    vals = _values(s["v_cache"][pt], ov, d).transpose(0, 1).flatten(1, 2)
    s["out"].copy_(torch.matmul(x, vals[:, None]).permute(2, 0, 1, 3).reshape(n, h * d))
    return {"out": s["out"]}


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt}[s["op"]](s)
    from realizar_b200 import ops
    if s["op"] == "append":
        ops.qk_norm_rope_append(s["qkv"], s["positions"], s["page_rows"], s["k_cache"], s["v_cache"], s["heads"], s["kv_heads"], s["head_dim"],
                                q_out=s["q_out"], q_norm_w=s["q_norm_w"], k_norm_w=s["k_norm_w"], eps=1e-6, rope_dim=s["rope_dim"],
                                rope_type=s["rope_type"], rope_table=s["rope_table"])
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if s["op"] == "decode":
        ops.attn_decode_launch(s["plan"])
        return {"out": s["out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    ops.attn_prefill(s["qkv"], s["out"], s["k_cache"], s["v_cache"], s["page_table"], s["rows"], s["pos0"], s["heads"], s["kv_heads"], s["head_dim"],
                     window=s["window"], scratch=s["scratch"])
    return {"out": s["out"]}


def work(case):
    c = case
    h, kvh, d = c["heads"], c["kv_heads"], c["head_dim"]
    row = 2 * kvh * _row_bytes(d)                                                                     # a token's bytes in the two caches
    if c["op"] == "append":
        live = c["rows"] - c["idle"]
        return {"bytes": live * ((2 * h + 2 * kvh) * d * 4 + row + 8 + 4 * c["rope_dim"]), "flops": live * (h + kvh) * d * 10}
    seen = lambda n: min(n, c["window"]) if c["window"] else n                                        # noqa: E731
    if c["op"] == "decode":
        keys = [seen(n) for n in _lengths(c)]
        return {"bytes": sum(keys) * row + c["batch"] * ((2 * h + 2 * kvh) * d * 4 + row) + sum(-(-n // PAGE) for n in keys) * 4,
                "flops": 4 * sum(keys) * h * d}
    total = c["pos0"] + c["rows"]
    keys = sum(seen(c["pos0"] + i + 1) for i in range(c["rows"]))
    read = min(total, c["window"] + c["rows"] - 1) if c["window"] else total
    return {"bytes": read * row + c["rows"] * h * d * 6, "flops": 4 * keys * h * d}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------
def _unpacked(cache, pages, d, keys):
    """Values of the listed pages in 64 bits, [kv heads, tokens, d], read by the order in which the codes lie."""
    flat = cache[pages].flatten(-2)
    n, kvh, full = flat.shape[0], flat.shape[1], d // 32
    if keys:
        words = flat[..., : 8 * d].reshape(n, kvh, PAGE, d // 8, 4)
        first = words[..., : 4 * full, :].reshape(n, kvh, PAGE, 4, full, 4).transpose(3, 4).reshape(n, kvh, PAGE, 4 * full, 4)
        byte = torch.cat([first, words[..., 4 * full:, :]], 3).reshape(n, kvh, PAGE, d // 2)
    else:
        byte = flat[..., : 256 * full].reshape(n, kvh, 2, 8, 4, full, 2, 2).permute(0, 1, 2, 4, 6, 5, 3, 7).reshape(n, kvh, PAGE, 16 * full)
        if d % 32:
            rest = flat[..., 256 * full: 8 * d].reshape(n, kvh, 8, 4, 2, 2).permute(0, 1, 4, 3, 5, 2).reshape(n, kvh, PAGE, 8)
            byte = torch.cat([byte, rest], -1)
    code = torch.empty(n, kvh, PAGE, d, dtype=torch.float64, device=DEV)
    code[..., 0::2], code[..., 1::2] = (byte % 16).double(), (byte // 16).double()
    meta = flat[..., 8 * d:].reshape(n, kvh, PAGE, 4).contiguous().view(torch.bfloat16).double()
    return (code * meta[..., 0:1] + meta[..., 1:2]).transpose(0, 1).reshape(kvh, n * PAGE, d)


def _heads64(s, what, w):
    """The query (0) or key (1) heads of every row after norm and rotation, in 64 bits, by turning each pair as a complex number."""
    h, kvh, d, r = s["heads"], s["kv_heads"], s["head_dim"], s["rope_dim"]
    x = s["qkv"][:, (0, h * d)[what]: (h * d, (h + kvh) * d)[what]].reshape(-1, (h, kvh)[what], d).double()
    if w is not None:
        x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / d + 1e-6) * w.double()
    turn = torch.view_as_complex(s["rope_table"].double())[s["positions"].clamp(min=0).long()][:, None]
    i = torch.arange(r // 2, device=DEV)
    first, second = (i, i + r // 2) if s["rope_type"] == 2 else (2 * i, 2 * i + 1)
    z = torch.complex(x[..., first], x[..., second]) * turn
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _row64(x):
    """What the cache returns for one row in 64 bits."""
    x = x.float().double()
    x = torch.nan_to_num(x, nan=0.0).clamp(-LIMIT, LIMIT)
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    scale, low = ((high - low) / 15).float().bfloat16().double(), low.bfloat16().double()
    return torch.where(scale > 0, ((x - low) / scale).round().clamp(0, 15) * scale, torch.zeros_like(x)) + low


def exact(case, seed):
    s = prepare(case, seed)
    h, kvh, d = s["heads"], s["kv_heads"], s["head_dim"]
    if s["op"] == "append":                                    # the caches hold whole numbers
        q = _heads64(s, 0, s["q_norm_w"]).flatten(1)
        return {"q": torch.where(s["positions"][:, None] >= 0, q, torch.zeros_like(q)), "k_cache": None, "v_cache": None}
    if s["op"] == "decode":
        q, k = _heads64(s, 0, s["q_norm_w"]), _row64(_heads64(s, 1, s["k_norm_w"]))
        v = _row64(s["qkv"][:, (h + kvh) * d:].reshape(-1, kvh, d).double())
        out = torch.zeros(q.shape[0], h * d, dtype=torch.float64, device=DEV)
        for b, p in enumerate(s["positions"].tolist()):
            lo = max(0, p + 1 - s["window"]) if s["window"] else 0
            pages = s["page_table"][b, lo // PAGE: p // PAGE + 1].long()
            ks, vs = _unpacked(s["k_cache"], pages, d, True), _unpacked(s["v_cache"], pages, d, False)
            at = p - lo // PAGE * PAGE
            ks[:, at], vs[:, at] = k[b], v[b]
            ks, vs = ks[:, lo % PAGE: at + 1], vs[:, lo % PAGE: at + 1]
            x = torch.softmax(torch.einsum("ngd,ntd->ngt", q[b].view(kvh, h // kvh, d), ks) / math.sqrt(d), -1)
            out[b] = torch.einsum("ngt,ntd->ngd", x, vs).reshape(-1)
        return {"out": out, "k_cache": None, "v_cache": None}
    n, pos0 = s["rows"], s["pos0"]
    ks, vs = (_unpacked(s[c], s["page_table"].long(), d, c == "k_cache")[:, : pos0 + n] for c in ("k_cache", "v_cache"))
    q = s["qkv"][:, : h * d].double().view(n, h, d)
    at, pos = torch.arange(pos0 + n, device=DEV), pos0 + torch.arange(n, device=DEV)[:, None]
    seen = (at <= pos) & ((at > pos - s["window"]) if s["window"] else True)
    out = torch.empty(n, h, d, dtype=torch.float64, device=DEV)
    for i in range(h):
        x = torch.where(seen, q[:, i] @ ks[i // (h // kvh)].t() / math.sqrt(d), -math.inf)
        out[:, i] = torch.softmax(x, -1) @ vs[i // (h // kvh)]
    return {"out": out.flatten(1)}
