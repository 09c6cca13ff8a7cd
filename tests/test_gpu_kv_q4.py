"""4-bit KV cache on the GPU: the fused norm + rotation + append, decode attention and prompt attention, each against a plain
computation in 64 bits, and the three together.

Tolerances.  Cached rows are compared bit for bit: the definition is in 64 bits and the kernels follow it exactly.  Rotated
queries go through about 3 roundings and a 7-level sum in 32 bits: 2e-6 of the norm covers 30 half-steps of 2^-24.  fp32
attention: operands are held to 22 bits (2^-23 each, query and probability), scores of size 10 carry 10 x 2^-22 into the
exponent, sums of up to some thousand terms add a few 2^-23: 1e-5 of the norm.  bf16 results add half a step of 2^-9 relative
to each value (rms 2^-9 / sqrt(3) = 1.1e-3 .. 2^-8 / 2), operands in 16 bits (fp16, 2^-12 each) stay well below: 4e-3 of the norm."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
LIMIT = 32768.0


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm().clamp(min=1e-300))


def _rope64(x, pos, table, rope_dim, rope_type):
    """x [n, heads, d] float64, table float32 (cos, sin)"""
    if not rope_dim:
        return x
    cs = table.double()[pos.clamp(min=0).long()][:, None]
    c, s = cs[..., 0], cs[..., 1]
    i = torch.arange(rope_dim // 2, device=x.device)
    p, q = (i, i + rope_dim // 2) if rope_type == 2 else (2 * i, 2 * i + 1)
    y = x.clone()
    y[..., p], y[..., q] = x[..., p] * c - x[..., q] * s, x[..., p] * s + x[..., q] * c
    return y


def _head64(x, w, pos, table, rope_dim, rope_type, eps=1e-6):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    return _rope64(x, pos, table, rope_dim, rope_type)


def _quant64(x):
    """What the cache returns for rows [..., d] (float32 arithmetic of the returned value, as kv_pages_to_float does it)."""
    x = x.float().double()
    x = torch.where(x.isnan(), 0.0, x).clamp(-LIMIT, LIMIT)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    sc, mn = ((hi - lo).float().double() / 15).float().bfloat16(), lo.float().bfloat16()
    code = torch.where(sc.double() > 0, ((x - mn.double()) / sc.double()).round().clamp(0, 15), 0.0)
    return code.float() * sc.float() + mn.float()


def _cache(n_pages, kvh, d, seed=0):
    from realizar_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    kv = ops.kv_cache_alloc(1, n_pages, kvh, d, "cuda", "q4")
    kv.copy_(torch.randint(0, 256, kv.shape, generator=g, device="cuda", dtype=torch.uint8))
    flat = kv.flatten(-2)
    shape = (2, 1, n_pages, kvh, 16)
    sc = 0.2 + 0.3 * torch.rand(shape, generator=g, device="cuda")
    mn = sc * (-7.5 + torch.randn(shape, generator=g, device="cuda"))
    flat[..., 8 * d:] = torch.stack([sc, mn], -1).bfloat16().view(torch.uint8).flatten(-2)
    return kv[0, 0], kv[1, 0]


def _gather(cache, pages, d, values, n):
    from realizar_b200 import ops
    return ops.kv_pages_to_float(cache[pages.long()], d, values).transpose(0, 1).flatten(1, 2)[:, :n].double()      # [kvh, n, d]


def _attend64(q, k, v, lo):
    """q [H, d], k / v [kvh, n, d]: attention to positions lo .. n-1"""
    kvh = k.shape[0]
    x = torch.einsum("hgd,hnd->hgn", q.view(kvh, -1, q.shape[-1]), k[:, lo:]) / math.sqrt(q.shape[-1])
    return torch.einsum("hgn,hnd->hgd", torch.softmax(x, -1), v[:, lo:]).reshape(-1)


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("d, h, kvh", [(64, 14, 2), (80, 4, 4), (96, 6, 1), (128, 16, 2)])
@pytest.mark.parametrize("rows, norm, rope_dim, rope_type, in_place", [(1, False, 32, 2, True), (37, True, -1, 2, False), (130, True, -1, 0, True), (19, False, 0, 0, False), (16, True, 50, 2, False)])
def test_append_matches_the_definition(cuda_device, d, h, kvh, rows, norm, rope_dim, rope_type, in_place):
    from realizar_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    rope_dim = d if rope_dim < 0 else rope_dim
    n_pages = rows // 16 + 4
    kc, vc = _cache(n_pages, kvh, d, seed=d)
    k0, v0 = kc.clone(), vc.clone()
    wide = torch.randn(rows, (h + 2 * kvh) * d + 24, generator=g, device="cuda") * 2                # row stride larger than the row
    qkv = wide[:, : (h + 2 * kvh) * d]
    first = 5                                                                                        # the rows start inside a page
    pos = (torch.arange(rows, device="cuda", dtype=torch.int32) + first)
    page_of = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    page_rows = page_of[(pos // 16).long()].contiguous()
    if rows > 8:
        pos[3] = -1; pos[rows - 2] = -1
    qw, kw = (1 + 0.2 * torch.randn(2, d, generator=g, device="cuda")).unbind(0) if norm else (None, None)
    table = ops.make_rope_table(rows + first, rope_dim, 1e4, "cuda") if rope_dim else None
    before = wide.clone()
    q_out = None if in_place else torch.full((rows, h * d), 7.0, device="cuda")
    if norm:
        qw, kw = qw.contiguous(), kw.contiguous()
    ops.qk_norm_rope_append(qkv, pos, page_rows, kc, vc, h, kvh, d, q_out=q_out, q_norm_w=qw, k_norm_w=kw, eps=1e-6, rope_dim=rope_dim, rope_type=rope_type, rope_table=table)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    q, k, v = before[:, : (h + 2 * kvh) * d].split([h * d, kvh * d, kvh * d], -1)
    live = pos >= 0
    want_q = _head64(q.view(rows, h, d), qw, pos, table, rope_dim, rope_type).flatten(1)
    got_q = wide[:, : h * d] if in_place else q_out
    assert _rel(got_q[live], want_q[live]) < 2e-6
    assert torch.equal(got_q[~live], (before[:, : h * d] if in_place else torch.full_like(got_q, 7.0))[~live])          # idle rows are left alone
    assert torch.equal(wide[:, h * d:], before[:, h * d:])
    if not in_place:
        assert torch.equal(wide, before)
    want_k, want_v = _quant64(_head64(k.view(rows, kvh, d), kw, pos, table, rope_dim, rope_type)), _quant64(v.reshape(rows, kvh, d).double())
    for cache, old, want, values in ((kc, k0, want_k, False), (vc, v0, want_v, True)):
        expect = ops.kv_pages_to_float(old, d, values)
        expect[page_rows[live].long(), :, (pos[live] % 16).long()] = want[live]
        assert torch.equal(ops.kv_pages_to_float(cache, d, values), expect)                             # every other row of the cache included


def test_append_special_values(cuda_device):
    """Constant rows, quotients that lie exactly on a border, NaN, infinities and values beyond the format's range."""
    from realizar_b200 import ops
    d, kvh = 64, 1
    kc, vc = _cache(2, kvh, d)
    rows = torch.zeros(8, 3 * d, device="cuda")
    v = rows[:, 2 * d:]
    v[0] = 3.25
    v[1, :32] = torch.arange(32, device="cuda") * 0.5; v[1, 32:] = 15.0; v[1, 31] = 15.0               # 0, 0.5, 1, ...: ties go to the even code
    v[2] = torch.randn(d, device="cuda"); v[2, 5] = float("nan")
    v[3] = torch.randn(d, device="cuda"); v[3, 0] = float("inf"); v[3, 9] = float("-inf")
    v[4] = torch.randn(d, device="cuda") * 1e30
    v[5] = torch.randn(d, device="cuda") * 1e-39                                                        # the scale is a subnormal number or 0
    v[6] = torch.randn(d, device="cuda") * 1e-3 + 100
    v[7, 0] = -1.0
    rows[:, d:2 * d] = v                                                                                # the same as keys, without norm and rotation
    pos, pages = torch.arange(8, device="cuda", dtype=torch.int32), torch.ones(8, device="cuda", dtype=torch.int32)
    ops.qk_norm_rope_append(rows, pos, pages, kc, vc, 1, kvh, d)
    want = _quant64(v.double())
    for cache, values in ((kc, False), (vc, True)):
        got = ops.kv_pages_to_float(cache[1], d, values)[0, :8]
        assert torch.equal(got, want)
        assert bool(got.isfinite().all()) and float(got.abs().max()) < 65504


def test_append_rejects_bad_pages_on_the_device(cuda_device):
    """A page id outside the cache: nothing of the row is cached, the other rows are, and the status word tells."""
    from realizar_b200 import ops
    d, kvh, h = 128, 2, 4
    kc, vc = _cache(3, kvh, d)
    k0 = kc.clone()
    qkv = torch.randn(3, (h + 2 * kvh) * d, device="cuda")
    pos, pages = torch.tensor([0, 1, 2], device="cuda", dtype=torch.int32), torch.tensor([3, 1, -1], device="cuda", dtype=torch.int32)
    q = torch.zeros(3, h * d, device="cuda")
    ops.device_error()
    ops.qk_norm_rope_append(qkv, pos, pages, kc, vc, h, kvh, d, q_out=q)
    torch.cuda.synchronize()
    assert ops.device_error() == 3405 and ops.device_error() == 0
    assert torch.equal(q, qkv[:, : h * d])
    assert torch.equal(kc[0], k0[0]) and torch.equal(kc[2], k0[2]) and not torch.equal(kc[1], k0[1])


def test_append_positions_beyond_the_table_use_theta(cuda_device):
    from realizar_b200 import ops
    d, kvh, h, n = 64, 1, 2, 3
    kc, vc = _cache(4, kvh, d)
    qkv = torch.randn(n, (h + 2 * kvh) * d, device="cuda")
    pos, pages = torch.tensor([2, 70_000, 1_000_003], device="cuda", dtype=torch.int32), torch.tensor([0, 1, 2], device="cuda", dtype=torch.int32)
    q = torch.zeros(n, h * d, device="cuda")
    ops.qk_norm_rope_append(qkv, pos, pages, kc, vc, h, kvh, d, q_out=q, rope_dim=d, rope_type=2, rope_theta=5e5, rope_table=ops.make_rope_table(3, d, 5e5, "cuda"))
    i = torch.arange(d // 2, dtype=torch.float64, device="cuda")
    ang = pos.double()[:, None] * torch.pow(torch.tensor(5e5, dtype=torch.float64, device="cuda"), -2 * i / d)
    c, s = ang.cos().float().double()[:, None], ang.sin().float().double()[:, None]
    x = qkv[:, : h * d].double().view(n, h, d)
    a, b = x[..., : d // 2], x[..., d // 2:]
    assert _rel(q, torch.cat([a * c - b * s, a * s + b * c], -1).flatten(1)) < 2e-6


# ------------------------------------------------------------------------------------------------ decode
def _decode(h, kvh, d, lens, seed, norm=False, rope_dim=0, rope_type=2, window=0, no_append=False, shared_table=False, garbage=True, scale_q=1.0):
    """One launch over sequences of the given lengths (new token included; 0: idle row) and what it should give."""
    from realizar_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, per = len(lens), max(1, -(-max(lens) // 16)) + 1
    n_pages = (1 if shared_table else B) * per + 2
    kc, vc = _cache(n_pages, kvh, d, seed)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    pt = order[:per].contiguous() if shared_table else order[: B * per].view(B, per).contiguous()
    if garbage:          # rows behind the last token of every sequence and pages that no sequence uses: bytes that decode to NaN and infinity
        for c in (kc, vc):
            flat = c.flatten(-2)
            for b, n in enumerate(lens):
                row = pt if shared_table else pt[b]
                last = max(lens) if shared_table else n
                meta = flat[row.long()][..., 8 * d:].unflatten(-1, (16, 4)).transpose(1, 2).flatten(0, 1)
                meta[last:] = 0xFF
                flat[row.long()[:, None, None], torch.arange(kvh, device="cuda")[None, :, None], torch.arange(8 * d, 8 * d + 64, device="cuda")] = \
                    meta.unflatten(0, (per, 16)).transpose(1, 2).flatten(-2)
            flat[order[(per if shared_table else B * per):].long()] = 0xFF
    qkv = torch.randn(B, (h + 2 * kvh) * d, generator=g, device="cuda")
    qkv[:, : h * d] *= scale_q
    pos = torch.tensor([n - 1 for n in lens], device="cuda", dtype=torch.int32)
    out = torch.full((B, h * d), 9.0, device="cuda")
    qw, kw = [w.contiguous() for w in (1 + 0.2 * torch.randn(2, d, generator=g, device="cuda")).unbind(0)] if norm else (None, None)
    table = ops.make_rope_table(max(lens) + 1, rope_dim, 1e4, "cuda") if rope_dim else None
    partial, counters = ops.attn_decode_scratch(B, h, 1, d, "cuda", kv_dtype="q4")
    p = ops.build_attn_decode_params(qkv, out, kc, vc, pos, pt, partial, counters, h, kvh, d, 1, B, rope_dim, rope_type, 1e4, 0, h * d, (h + kvh) * d, qw, kw, 1e-6,
                                     window=window, rope_table=table, no_append=no_append, shared_table=shared_table)
    keep = (qkv, out, kc, vc, pos, pt, partial, counters, qw, kw, table)
    k0, v0 = kc.clone(), vc.clone()

    def check(launch=True):
        if launch:
            ops.attn_decode_launch(p)
        torch.cuda.synchronize()
        assert ops.device_error() == 0
        q, k, v = qkv.split([h * d, kvh * d, kvh * d], -1)
        q = _head64(q.view(B, h, d), qw, pos, table, rope_dim, rope_type)
        k, v = _quant64(_head64(k.view(B, kvh, d), kw, pos, table, rope_dim, rope_type)), _quant64(v.reshape(B, kvh, d).double())
        worst = 0.0
        for b, p1 in enumerate(pos.tolist()):
            if p1 < 0:
                assert torch.equal(out[b], torch.full_like(out[b], 9.0))
                continue
            row = pt if shared_table else pt[b]
            ks, vs = _gather(kc, row, d, False, p1 + 1), _gather(vc, row, d, True, p1 + 1)
            if not no_append:
                assert torch.equal(ks[:, p1].float(), k[b]) and torch.equal(vs[:, p1].float(), v[b])        # the appended rows, bit for bit
            want = _attend64(q[b], ks, vs, max(0, p1 + 1 - window) if window else 0)
            worst = max(worst, _rel(out[b], want))
        touched = [(int((pt if shared_table else pt[b])[p1 // 16]), p1 % 16) for b, p1 in enumerate(pos.tolist()) if p1 >= 0 and not no_append]
        for c, old in ((kc, k0), (vc, v0)):                                                                  # nothing else of the cache changed
            same = (ops.kv_pages_to_float(c, d, c is vc).nan_to_num() == ops.kv_pages_to_float(old, d, c is vc).nan_to_num()).all(-1).all(1)
            for pg, s in touched:
                same[pg, s] = True
            assert bool(same.all())
        assert worst < 1e-5, worst
    check.params, check.keep = p, keep
    return check


@pytest.mark.parametrize("h, kvh, d", [(8, 8, 80), (14, 2, 64), (6, 1, 96), (32, 8, 128), (12, 1, 64), (20, 1, 128), (1, 1, 80)])
@pytest.mark.parametrize("lens", [[1], [17, 1, 16, 0, 300, 47], [1000]])
def test_decode_attention(cuda_device, h, kvh, d, lens):
    _decode(h, kvh, d, lens, seed=h + d + len(lens), norm=True, rope_dim=d, rope_type=2)()


@pytest.mark.parametrize("kw", [dict(window=1), dict(window=16), dict(window=33, rope_dim=32, rope_type=0), dict(no_append=True), dict(no_append=True, shared_table=True),
                                dict(norm=True), dict(scale_q=30.0), dict(scale_q=0.0), dict(window=5000, rope_dim=64)])
def test_decode_attention_options(cuda_device, kw):
    lens = [64, 31, 64, 5] if kw.get("shared_table") else [97, 1, 32, 700, 33]
    _decode(8, 2, 128, lens, seed=5, **kw)()


@pytest.mark.parametrize("B, n", [(1, 40000), (1, 131072), (200, 70), (3, 5000), (600, 3)])
def test_decode_attention_divides_any_batch(cuda_device, B, n):
    _decode(8, 4, 64, [max(1, n - 13 * (b % 5)) for b in range(B)], seed=B, rope_dim=64)()


def test_decode_wide_ranges_of_scales(cuda_device):
    """Rows whose scales differ by many orders of magnitude, all-constant rows first, one row that takes all of the attention."""
    from realizar_b200 import ops
    h, kvh, d, n = 4, 1, 64, 200
    for kind in ("constant first", "growing", "shrinking", "peaked"):
        check = _decode(h, kvh, d, [n], seed=3, no_append=True)
        qkv, out, kc, vc, pos, pt = check.keep[:6]
        flat = vc.flatten(-2)
        meta = torch.zeros(pt.numel() * 16, 2, device="cuda")
        i = torch.arange(pt.numel() * 16, device="cuda").float()
        meta[:, 0] = {"constant first": torch.where(i < 64, 0.0, 1e-6), "growing": torch.exp2(i / 8 - 20), "shrinking": torch.exp2(5 - i / 8), "peaked": 0.3 + 0 * i}[kind]
        meta[:, 1] = -7.5 * meta[:, 0]
        flat[pt[0].long(), 0, 8 * d:] = meta.bfloat16().view(torch.uint8).view(-1, 64)
        if kind == "peaked":
            kflat = kc.flatten(-2)
            km = kflat[pt[0].long(), 0, 8 * d:].contiguous().view(torch.bfloat16).view(-1, 2)
            km[150] *= 40
            kflat[pt[0].long(), 0, 8 * d:] = km.view(torch.uint8).view(-1, 64)
        ops.attn_decode_launch(check.params)
        q = qkv[0, : h * d].double().view(h, d)
        want = _attend64(q, _gather(kc, pt[0], d, False, n), _gather(vc, pt[0], d, True, n), 0)
        assert _rel(out[0], want) < 1e-5, kind


@pytest.mark.parametrize("h, kvh, d, grow", [(8, 2, 64, True), (14, 2, 80, True), (4, 2, 96, False), (6, 1, 128, True), (16, 2, 128, False)])
def test_decode_long_shares(cuda_device, h, kvh, d, grow):
    """Many rows over the same long context, so that a warp goes through dozens of pages: its sums leave the registers on the way.  With
    ``grow``, scores and values grow along the context: the running maximum and the values' power of two move after that.

    Scores reach 20 in powers of two and are rounded some three times: 3 x 20 x 2^-24 x ln 2 = 2.5e-6, and the sums add less than 2e-6."""
    from realizar_b200 import ops
    B, n = 64 if kvh == 2 else 128, 6000
    check = _decode(h, kvh, d, [n - 7 * (b % 3) for b in range(B)], seed=d + h, no_append=True, shared_table=True, garbage=False)
    qkv, out, kc, vc, pos, pt = check.keep[:6]
    if grow:
        i = torch.arange(pt.numel() * 16, device="cuda").float()[:, None]
        for c, factor in ((kc, torch.exp2(i / n)), (vc, torch.exp2(i / 400 - 8))):
            flat = c.flatten(-2)
            for k in range(kvh):
                meta = flat[pt.long(), k, 8 * d:].contiguous().view(torch.bfloat16).view(-1, 2).float()
                flat[pt.long(), k, 8 * d:] = (meta * factor).bfloat16().view(torch.uint8).view(-1, 64)
    ops.attn_decode_launch(check.params)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    ks, vs = _gather(kc, pt, d, False, n), _gather(vc, pt, d, True, n)
    for b in range(0, B, 5):
        p1 = int(pos[b]) + 1
        assert _rel(out[b], _attend64(qkv[b, : h * d].double().view(h, d), ks[:, :p1], vs[:, :p1], 0)) < 1e-5, b


def test_decode_device_checks(cuda_device):
    """A position beyond its page-table row and a page id outside the cache set the status word; the other sequences are right."""
    from realizar_b200 import ops
    check = _decode(8, 2, 64, [40, 50, 60], seed=1, rope_dim=64)
    qkv, out, kc, vc, pos, pt = check.keep[:6]
    keep = pos.clone()
    pos[1] = pt.shape[1] * 16
    ops.device_error()
    ops.attn_decode_launch(check.params)
    torch.cuda.synchronize()
    assert ops.device_error() == 3311 and bool((out[1] == 9.0).all()) and not bool((out[0] == 9.0).any())
    pos.copy_(keep)
    good = pt[1, 0].clone()
    pt[1, 0] = kc.shape[0]
    ops.attn_decode_launch(check.params)
    torch.cuda.synchronize()
    assert ops.device_error() == 3312
    pt[1, 0] = good
    check()


def test_decode_graph_replays_with_new_positions_and_shares_scratch(cuda_device):
    """Two captured graphs with one workspace, replayed in turn while the sequences grow."""
    a = _decode(8, 2, 128, [250, 3, 90], seed=2, rope_dim=128)
    b = _decode(8, 2, 128, [60], seed=4, rope_dim=128)
    b.params.partial, b.params.counters = a.params.partial, a.params.counters
    from realizar_b200 import ops
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.attn_decode_launch(a.params); ops.attn_decode_launch(b.params)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.attn_decode_launch(c.params)
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
    a(launch=False); b(launch=False)
    first = a.keep[1].clone()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(a.keep[1], first)                       # the same bits every time
    a.keep[4][1] = 1                                           # a shorter sequence in the same graph
    graphs[0].replay(); graphs[1].replay()
    torch.cuda.synchronize()
    row, p1 = a.keep[5][1], 1
    q = _head64(a.keep[0][1:2, : 8 * 128].view(1, 8, 128), None, a.keep[4][1:2], a.keep[10], 128, 2)[0]
    want = _attend64(q, _gather(a.keep[2], row, 128, False, 2), _gather(a.keep[3], row, 128, True, 2), 0)
    assert _rel(a.keep[1][1], want) < 1e-5


# ------------------------------------------------------------------------------------------------ prompt
def _prompt(h, kvh, d, rows, pos0, window=0, out_dtype=torch.bfloat16, with_scratch=True, dev_pos=False, tol=4e-3):
    from realizar_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(rows + pos0 + d)
    total = pos0 + rows
    per = -(-total // 16) + 1
    kc, vc = _cache(per + 2, kvh, d, seed=rows)
    pt = torch.randperm(per + 2, generator=g, device="cuda").to(torch.int32)[:per].contiguous()
    for c in (kc, vc):                                          # behind the last token: bytes that decode to NaN
        flat = c.flatten(-2)
        meta = flat[pt.long()][..., 8 * d:].unflatten(-1, (16, 4)).transpose(1, 2).flatten(0, 1)
        meta[total:] = 0xFF
        flat[pt.long()[:, None, None], torch.arange(kvh, device="cuda")[None, :, None], torch.arange(8 * d, 8 * d + 64, device="cuda")] = \
            meta.unflatten(0, (per, 16)).transpose(1, 2).flatten(-2)
    qkv = torch.randn(rows + 2, (h + 2 * kvh) * d, generator=g, device="cuda")
    out = torch.full((rows + 2, h * d + 8), 9.0, device="cuda", dtype=out_dtype)
    scratch = ops.attn_prefill_scratch(rows, h, kvh, d, "cuda") if with_scratch else None
    pd = torch.tensor([pos0], device="cuda", dtype=torch.int32) if dev_pos else None
    for _ in range(2):                                          # twice: the workspace keeps nothing
        ops.attn_prefill(qkv, out[:, 8:], kc, vc, pt, rows, 0 if dev_pos else pos0, h, kvh, d, window=window, pos0_dev=pd, scratch=scratch)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    assert bool((out[:, :8] == 9.0).all()) and bool((out[rows:] == 9.0).all())
    ks, vs = _gather(kc, pt, d, False, total), _gather(vc, pt, d, True, total)
    at, pos = torch.arange(total, device="cuda"), pos0 + torch.arange(rows, device="cuda")[:, None]
    seen = (at <= pos) & ((at > pos - window) if window else True)
    q = qkv[:rows, : h * d].double().view(rows, kvh, h // kvh, d)
    x = torch.where(seen[:, None, None], torch.einsum("rkgd,knd->rkgn", q, ks) / math.sqrt(d), -math.inf)
    want = torch.einsum("rkgn,knd->rkgd", torch.softmax(x, -1), vs).reshape(rows, h * d)
    got = out[:rows, 8:]
    assert _rel(got, want) < tol, _rel(got, want)
    per_row = ((got.double() - want).norm(dim=-1) / want.norm(dim=-1)).max()
    assert float(per_row) < 3 * tol, float(per_row)


@pytest.mark.parametrize("h, kvh, d", [(4, 4, 80), (14, 2, 64), (6, 1, 96), (16, 4, 128), (12, 1, 64), (5, 5, 128)])
@pytest.mark.parametrize("rows, pos0", [(1, 0), (16, 0), (77, 1337), (130, 31), (300, 0)])
def test_prompt_attention(cuda_device, h, kvh, d, rows, pos0):
    _prompt(h, kvh, d, rows, pos0)


@pytest.mark.parametrize("kw", [dict(window=1), dict(window=50), dict(window=300), dict(with_scratch=False), dict(dev_pos=True), dict(out_dtype=torch.float32)])
def test_prompt_attention_options(cuda_device, kw):
    _prompt(8, 2, 128, 150, 420, **kw)


def test_prompt_attention_long(cuda_device):
    _prompt(8, 2, 128, 40, 9000)
    _prompt(8, 1, 64, 1100, 1500)


@pytest.mark.parametrize("h, kvh, d, rows, pos0, kw", [
    (8, 4, 64, 4999, 0, dict(window=2000)), (16, 16, 80, 1700, 5995, {}), (8, 8, 96, 3600, 700, dict(dev_pos=True, window=900)), (24, 8, 128, 1501, 3333, dict(out_dtype=torch.float32))])
def test_prompt_attention_divided_evenly(cuda_device, h, kvh, d, rows, pos0, kw):
    """More row tiles than SMs, or a number that leaves many idle: shares that begin and end inside row tiles, tiles with one group of rows."""
    _prompt(h, kvh, d, rows, pos0, **kw)


@pytest.mark.parametrize("h, kvh, d, rows, pos0, kw", [
    (64, 1, 128, 3, 700, {}), (300, 1, 64, 2, 100, {}), (160, 160, 64, 9, 40, {}), (160, 160, 80, 300, 5, dict(with_scratch=False)), (2, 1, 128, 129, 5000, {}),
    (18, 18, 64, 100, 900, {}), (19, 19, 128, 200, 1500, dict(window=700)), (1, 1, 64, 1, 60000, {}), (1, 1, 64, 1, 60000, dict(with_scratch=False)),
    (4, 4, 128, 129, 2047, {}), (74, 74, 64, 16, 5000, {}), (75, 75, 64, 16, 5000, {})])
def test_prompt_attention_at_the_borders_of_the_split(cuda_device, h, kvh, d, rows, pos0, kw):
    """More query heads than rows of a tile, more kv heads than SMs, one row over a long context, row tiles that just fill or just miss two
    CTAs each, a second group of one row."""
    _prompt(h, kvh, d, rows, pos0, **kw)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 600])
def test_prompt_attention_window_beyond_the_positions(cuda_device, window):
    _prompt(4, 2, 64, 90, 500, window=window)


def test_prompt_attention_rows_on_odd_addresses(cuda_device):
    """Query rows that start on 4-byte boundaries only."""
    from realizar_b200 import ops
    h, kvh, d, n = 6, 2, 80, 70
    kc, vc = _cache(6, kvh, d)
    pt = torch.arange(6, device="cuda", dtype=torch.int32)
    qkv = torch.randn(n, (h + 2 * kvh) * d, device="cuda")
    odd = torch.zeros(n, (h + 2 * kvh) * d + 3, device="cuda")[:, 1:]
    odd[:, :qkv.shape[1]] = qkv
    a, b = torch.empty(2, n, h * d, device="cuda")
    ops.attn_prefill(qkv, a, kc, vc, pt, n, 5, h, kvh, d)
    ops.attn_prefill(odd, b, kc, vc, pt, n, 5, h, kvh, d)
    assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["constant first", "growing", "shrinking"])
def test_prompt_wide_ranges_of_scales(cuda_device, kind):
    """Values whose scales differ by many orders of magnitude: the operands' power of two moves with them."""
    from realizar_b200 import ops
    h, kvh, d, n, rows = 4, 1, 64, 400, 60
    kc, vc = _cache(26, kvh, d)
    pt = torch.randperm(26, device="cuda").to(torch.int32)[:25].contiguous()
    i = torch.arange(400, device="cuda").float()
    sc = {"constant first": torch.where(i < 200, 0.0, 1e-6), "growing": torch.exp2(i / 16 - 20), "shrinking": torch.exp2(5 - i / 16)}[kind]
    vc.flatten(-2)[pt.long(), 0, 8 * d:] = torch.stack([sc, -7.5 * sc], -1).bfloat16().view(torch.uint8).view(-1, 64)
    qkv = torch.randn(rows, (h + 2 * kvh) * d, device="cuda")
    ks, vs = _gather(kc, pt, d, False, n), _gather(vc, pt, d, True, n)
    for scratch in (None, ops.attn_prefill_scratch(rows, h, kvh, d, "cuda")):
        out = torch.empty(rows, h * d, device="cuda")
        ops.attn_prefill(qkv, out, kc, vc, pt, rows, n - rows, h, kvh, d, scratch=scratch)
        for r in range(0, rows, 7):
            p1 = n - rows + r + 1
            assert _rel(out[r], _attend64(qkv[r, : h * d].double().view(h, d), ks[:, :p1], vs[:, :p1], 0)) < 4e-3, r


def test_prompt_device_checks(cuda_device):
    """Rows beyond the page table are left alone, a page id outside the cache reads page 0; the status word tells of both."""
    from realizar_b200 import ops
    h, kvh, d, n = 8, 2, 128, 40
    kc, vc = _cache(5, kvh, d)
    pt = torch.tensor([3, 0, 2, 1], device="cuda", dtype=torch.int32)
    qkv, out = torch.randn(n, (h + 2 * kvh) * d, device="cuda"), torch.full((n, h * d), 9.0, device="cuda")
    ops.device_error()
    for first in (25, -1, 2 ** 31 - 8):
        ops.attn_prefill(qkv, out, kc, vc, pt, n, 0, h, kvh, d, pos0_dev=torch.tensor([first], device="cuda", dtype=torch.int32))
        torch.cuda.synchronize()
        assert ops.device_error() == 3114 and ops.device_error() == 0 and bool((out == 9.0).all())
    ops.attn_prefill(qkv, out, kc, vc, pt, n, 0, h, kvh, d, pos0_dev=torch.tensor([24], device="cuda", dtype=torch.int32))
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    for bad in (5, -3):
        ops.attn_prefill(qkv, out, kc, vc, torch.tensor([3, bad, 2, 1], device="cuda", dtype=torch.int32), n, 24, h, kvh, d)
        torch.cuda.synchronize()
        want = torch.empty_like(out)
        assert ops.device_error() == 3113
        ops.attn_prefill(qkv, want, kc, vc, pt, n, 24, h, kvh, d)
        assert torch.equal(out, want)


def test_prompt_scratch_of_other_sizes(cuda_device):
    """A workspace that is too small is not used, a larger one is; both leave it as it was for the next call."""
    from realizar_b200 import ops
    small, large = ops.attn_prefill_scratch(64, 4, 1, 64, "cuda"), ops.attn_prefill_scratch(64, 4, 1, 128, "cuda")
    res = []
    for d in (128, 64, 128):
        kc, vc = _cache(60, 1, d, seed=1)
        pt, qkv = torch.arange(60, device="cuda", dtype=torch.int32), torch.randn(64, 6 * d, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
        outs = [torch.empty(64, 4 * d, device="cuda") for _ in range(3)]
        for o, s in zip(outs, (None, small, large)):
            ops.attn_prefill(qkv, o, kc, vc, pt, 64, 800, 4, 1, d, scratch=s)
        assert ops.device_error() == 0
        assert _rel(outs[1], outs[0]) < 1e-3 and _rel(outs[2], outs[0]) < 1e-3          # P is rounded to fp16 (2^-12) against the maximum of other parts
        res.append(outs)
    assert torch.equal(res[0][2], res[2][2])


# ------------------------------------------------------------------------------------------------ together
def test_captured_append_and_prompt_replay_at_other_positions(cuda_device):
    """A chunk's append and attention in one graph: positions, pages and the first position are read on the device.  Two graphs share a workspace."""
    from realizar_b200 import ops
    h, kvh, d, n = 8, 2, 128, 32
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(96, (h + 2 * kvh) * d, generator=g, device="cuda")
    table, pt = ops.make_rope_table(128, d, 1e4, "cuda"), torch.tensor([4, 1, 6, 0, 5, 2], device="cuda", dtype=torch.int32)
    scratch = ops.attn_prefill_scratch(n, h, kvh, d, "cuda")
    caches = [ops.kv_cache_alloc(1, 7, kvh, d, "cuda", "q4")[:, 0] for _ in range(3)]

    def chunk(c, first, qkv, pos, pages, p0, out):
        qkv.copy_(x[first:first + n])
        pos.copy_(torch.arange(first, first + n, dtype=torch.int32)); pages.copy_(pt[(pos // 16).long()]); p0.fill_(first)

    def launches(c, qkv, pos, pages, p0, out):
        ops.qk_norm_rope_append(qkv, pos, pages, caches[c][0], caches[c][1], h, kvh, d, rope_dim=d, rope_type=2, rope_table=table)
        ops.attn_prefill(qkv, out, caches[c][0], caches[c][1], pt, n, 0, h, kvh, d, pos0_dev=p0, scratch=scratch)

    bufs = [(torch.empty(n, x.shape[1], device="cuda"), torch.empty(n, device="cuda", dtype=torch.int32), torch.empty(n, device="cuda", dtype=torch.int32),
             torch.zeros(1, device="cuda", dtype=torch.int32), torch.empty(n, h * d, device="cuda", dtype=torch.bfloat16)) for _ in range(3)]
    graphs = []
    for c in (0, 1):
        chunk(c, 0, *bufs[c])
        launches(c, *bufs[c])
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[c]):
            launches(c, *bufs[c])
    for c in range(3):
        caches[c].zero_()
    for first in (0, 32, 64):
        for c in range(3):
            chunk(c, first, *bufs[c])
        for c in (0, 1):
            graphs[c].replay()
        launches(2, *bufs[2])
        torch.cuda.synchronize()
        assert ops.device_error() == 0
        for c in (0, 1):
            assert torch.equal(bufs[c][4], bufs[2][4]) and torch.equal(caches[c], caches[2])


def test_prompts_on_two_streams_with_their_own_workspaces(cuda_device):
    from realizar_b200 import ops
    h, kvh, d = 8, 2, 64
    jobs = []
    for i, (n, first) in enumerate(((50, 900), (300, 700))):
        kc, vc = _cache(64, kvh, d, seed=i)
        qkv = torch.randn(n, (h + 2 * kvh) * d, device="cuda")
        a = (kc, vc, torch.randperm(64, device="cuda").to(torch.int32), n, first, h, kvh, d)
        want, scratch = torch.empty(n, h * d, device="cuda"), ops.attn_prefill_scratch(n, h, kvh, d, "cuda")
        ops.attn_prefill(qkv, want, *a, scratch=scratch)
        jobs.append((qkv, torch.empty_like(want), a, scratch, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for qkv, out, a, scratch, _, stream in jobs:
            with torch.cuda.stream(stream):
                ops.attn_prefill(qkv, out, *a, scratch=scratch)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    for _, out, _, _, want, _ in jobs:
        assert torch.equal(out, want)


def test_decode_static_entry_point(cuda_device):
    """The entry point with built-in scratch takes 4-bit caches too, twice in a row."""
    import ctypes
    from realizar_b200 import ops
    fn = ops.lib().rlz_attn_decode_static
    fn.argtypes, fn.restype = [ctypes.c_void_p, ctypes.c_void_p], ctypes.c_int
    check = _decode(8, 2, 128, [3000, 17], seed=6, rope_dim=128)
    check()
    want = check.keep[1].clone()
    for _ in range(2):
        check.keep[1].fill_(9.0)
        assert fn(ctypes.addressof(check.params), torch.cuda.current_stream().cuda_stream) == 0
        check(launch=False)
        assert torch.equal(check.keep[1], want)


def test_append_prompt_decode_as_a_serving_pass(cuda_device):
    """A prompt in two chunks and then single tokens, all through the cache, against attention in 64 bits over the values the cache holds;
    the rows a prompt pass writes and those a decode step writes are the same bits."""
    from realizar_b200 import ops
    h, kvh, d, n, steps = 8, 2, 128, 90, 5
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(n + steps, (h + 2 * kvh) * d, generator=g, device="cuda")
    qw, kw = [w.contiguous() for w in (1 + 0.2 * torch.randn(2, d, generator=g, device="cuda")).unbind(0)]
    table = ops.make_rope_table(256, d, 1e4, "cuda")
    pt = torch.tensor([[5, 2, 7, 0, 3, 6]], device="cuda", dtype=torch.int32)
    caches = [ops.kv_cache_alloc(1, 8, kvh, d, "cuda", "q4")[:, 0] for _ in range(2)]
    kc, vc = caches[0]
    pos = torch.arange(n + steps, device="cuda", dtype=torch.int32)
    rows = pt[0, (pos // 16).long()].contiguous()
    kw_args = dict(q_norm_w=qw, k_norm_w=kw, eps=1e-6, rope_dim=d, rope_type=2, rope_table=table)
    ops.qk_norm_rope_append(x, pos, rows, caches[1][0], caches[1][1], h, kvh, d, q_out=torch.empty(n + steps, h * d, device="cuda"), **kw_args)
    outs = []
    scratch = ops.attn_prefill_scratch(64, h, kvh, d, "cuda")
    for c0, c1 in ((0, 64), (64, n)):
        chunk, out = x[c0:c1].clone(), torch.empty(c1 - c0, h * d, device="cuda", dtype=torch.bfloat16)
        ops.qk_norm_rope_append(chunk, pos[c0:c1], rows[c0:c1], kc, vc, h, kvh, d, **kw_args)
        ops.attn_prefill(chunk, out, kc, vc, pt[0], c1 - c0, c0, h, kvh, d, scratch=scratch)
        outs.append(out.float())
    partial, counters = ops.attn_decode_scratch(1, h, 1, d, "cuda", kv_dtype="q4")
    for i in range(n, n + steps):
        out = torch.empty(1, h * d, device="cuda")
        p = ops.build_attn_decode_params(x[i:i + 1], out, kc, vc, pos[i:i + 1], pt, partial, counters, h, kvh, d, 1, 1, d, 2, 1e4, 0, h * d, (h + kvh) * d, qw, kw, 1e-6,
                                         rope_table=table)
        ops.attn_decode_launch(p)
        outs.append(out)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    assert torch.equal(caches[0], caches[1])
    got = torch.cat(outs)
    q = _head64(x[:, : h * d].view(-1, h, d), qw, pos, table, d, 2)
    ks, vs = _gather(kc, pt[0], d, False, n + steps), _gather(vc, pt[0], d, True, n + steps)
    for i in range(n + steps):
        assert _rel(got[i], _attend64(q[i], ks[:, : i + 1], vs[:, : i + 1], 0)) < (4e-3 * 3 if i < n else 1e-5), i


def test_two_streams_with_their_own_workspaces(cuda_device):
    a, b = _decode(8, 2, 128, [2000, 900], seed=8, rope_dim=128), _decode(14, 2, 64, [1500], seed=9, rope_dim=64)
    from realizar_b200 import ops
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for s, c in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                ops.attn_decode_launch(c.params)
    a(launch=False); b(launch=False)


@pytest.mark.parametrize("name", ["llama", "phi2"])
def test_engine_serves_from_the_4_bit_cache(cuda_device, name):
    """Prefill in chunks, decode steps, a batch and a snapshot over kv_dtype='q4': logits stay near those of the bf16 cache, the
    cache takes (d / 2 + 4) / 2 d of the memory and results do not depend on the path that wrote it.

    How near: a row of 64 or 80 normal values spans about 4.7 sigma, a step is 4.7 / 15 = 0.31 sigma, so every cached value is off by
    0.31 / sqrt(12) = 0.09 sigma.  Scores q.k / sqrt(d) of these weights have a spread of about 1.3 and are off by 0.12, which moves the
    weights by 12%; with the 9% of the values that is 15% to each attention output.  A gated layer (a product of two) doubles it and two
    layers add up: at most 2 x 15% x sqrt(2) = 42% of the logits if nothing came past the attention, a cosine of 1 / sqrt(1 + 0.42^2) = 0.92."""
    from test_gpu_engine import _cos, _kq_llama, small_phi2
    from realizar_b200.models.weights import synthetic_weights
    from realizar_b200.runtime.engine import DecodeEngine, EngineConfig
    cfg = _kq_llama() if name == "llama" else small_phi2()
    w = synthetic_weights(cfg, seed=21, std=0.05, **({} if name == "llama" else {"scheme": "Q4_K_M"}))
    toks = [int(t) for t in np.random.default_rng(8).integers(0, cfg.vocab_size, 90)]
    res = {}
    for kd in ("bf16", "q4"):
        eng = DecodeEngine(w, EngineConfig(max_batch=2, max_seq_len=160, greedy_only=True, kv_dtype=kd, prefill_chunk=64))
        eng.open_slot(0, 128)
        nxt = eng.prefill(0, toks)
        logits = [eng.logits_of_last_step(0).float().cpu().numpy()]
        for t in (5, 17, 3):
            eng.feed({0: t})
            logits.append(eng.logits_of_last_step(0).float().cpu().numpy())
        res[kd] = (logits, eng.memory_report()["kv_bytes"])
        if kd == "q4":
            snap = eng.snapshot_kv(0)
            eng.open_slot(1, 128)
            eng.restore_kv(1, snap)
            a, b = (eng.feed({s: 9}) is not None and eng.logits_of_last_step(s).float().cpu().numpy() for s in (0, 1))
            assert _cos(a, b) > 0.99999
            eng.check_health()
        eng.close()
    hd = cfg.head_dim
    assert res["q4"][1] * 2 * hd == res["bf16"][1] * (hd // 2 + 4)
    for a, b in zip(res["bf16"][0], res["q4"][0]):
        assert _cos(a, b) > 0.9, _cos(a, b)


# ------------------------------------------------------------------------------------------------ a key that takes nearly all of the weight
def _one_key_takes(share, kc, vc, pt, n, h, kvh, d, rows, seed=0):
    """Query rows whose scores have a spread of about 1 over the first ``n`` rows of the table, but for the row at position 0: its key is
    a constant that every query scores alike, so that it takes ``share`` of the weight, and its value row is zero.  What is left of
    the result is the sum of the small weights.  Returns the queries and the constant."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    total = 0.4                                                   # sum(q) / sqrt(d)
    q = 0.6 * torch.randn(rows, h, d, generator=g, device="cuda")
    q += total / math.sqrt(d) - q.mean(-1, keepdim=True)
    top = (math.log(share / (1 - share)) + math.log(n) + 0.5) / total
    for c, low in ((kc, top), (vc, 0.0)):
        flat = c.flatten(-2)
        flat[int(pt[0]), :, 8 * d: 8 * d + 4] = torch.tensor([0.0, low], device="cuda").bfloat16().view(torch.uint8)
    return q.reshape(rows, h * d), top


@pytest.mark.parametrize("h, kvh, d, share", [(8, 2, 64, 0.97), (14, 2, 128, 0.97), (8, 2, 80, 0.999), (6, 1, 96, 0.999)])
def test_decode_with_one_key_that_takes_the_weight(cuda_device, h, kvh, d, share):
    """The file's 1e-5 where the largest weight belongs to a value of zero, and what the rounding of the queries does to that weight.  A weight
    times its value's scale is held to 22 bits of itself, so the small ones count as exactly as large ones.

    The key of the large weight is ``top`` in all dims, and its score the sum of top q_i / sqrt(d), in which the q_i cancel but their roundings
    to integers do not: half a step is at most 2^-23 x 128 / 127 of the row's largest |q|, in the root mean square 1 / sqrt(3) of that.  The
    score is off by top x max|q| x 2^-23 x 1.008 / sqrt(3), and the result by that fraction of itself."""
    from realizar_b200 import ops
    B, n = 64 if kvh == 2 else 128, 32768
    check = _decode(h, kvh, d, [n] * B, seed=d, no_append=True, shared_table=True, garbage=False)
    qkv, out, kc, vc, pos, pt = check.keep[:6]
    qkv[:, : h * d], top = _one_key_takes(share, kc, vc, pt, n, h, kvh, d, B)
    ops.attn_decode_launch(check.params)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    ks, vs = _gather(kc, pt, d, False, n), _gather(vc, pt, d, True, n)
    room = top * float(qkv[:, : h * d].abs().max()) * 2.0 ** -23 * 1.008 / math.sqrt(3)
    worst = max(_rel(out[b], _attend64(qkv[b, : h * d].double().view(h, d), ks, vs, 0)) for b in range(0, B, 5))
    assert worst < 1e-5 + room, worst


@pytest.mark.parametrize("d, share, with_scratch", [(64, 0.97, False), (128, 0.97, True), (80, 0.999, False), (96, 0.999, True)])
def test_prompt_with_one_key_that_takes_the_weight(cuda_device, d, share, with_scratch):
    """The file's 4e-3 where the largest weight belongs to a value of zero, and what the rounding of the queries does to that weight.  The row
    tiles leave no CTAs for a cluster (without a workspace a CTA takes all keys of a row), so that the small weights are held against the
    large one.

    The key of the large weight is ``top`` in all dims, and its score the sum of top q_i / sqrt(d), in which the q_i (rms 0.6) cancel but their
    roundings do not: each q_i is off by at most half a step of fp16, 2^-11 |q_i|, in the mean square by at most 2^-11 |q_i| / sqrt(3).  The score is
    off by top x 0.6 x 2^-11 / sqrt(3) in the root mean square over the heads, the weight and with it the sum of the weights by that fraction of
    itself, and the result by the same."""
    from realizar_b200 import ops
    kvh, rows, n = 80, 8, 32768
    per = n // 16
    kc, vc = _cache(per + 2, kvh, d, seed=d)
    pt = torch.randperm(per + 2, device="cuda", generator=torch.Generator(device="cuda").manual_seed(d)).to(torch.int32)[:per].contiguous()
    qkv = torch.zeros(rows, 3 * kvh * d, device="cuda")
    qkv[:, : kvh * d], top = _one_key_takes(share, kc, vc, pt, n, kvh, kvh, d, rows)
    out = torch.empty(rows, kvh * d, device="cuda")
    scratch = ops.attn_prefill_scratch(rows, kvh, kvh, d, "cuda") if with_scratch else None
    ops.attn_prefill(qkv, out, kc, vc, pt, rows, n - rows, kvh, kvh, d, scratch=scratch)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    ks, vs = _gather(kc, pt, d, False, n), _gather(vc, pt, d, True, n)
    worst = max(_rel(out[r], _attend64(qkv[r, : kvh * d].double().view(kvh, d), ks[:, : n - rows + r + 1], vs[:, : n - rows + r + 1], 0)) for r in range(rows))
    assert worst < 4e-3 + top * 0.6 * 2.0 ** -11 / math.sqrt(3), worst


def test_append_and_decode_take_eps_alike(cuda_device):
    """Keys so small that eps decides their norm, of them those that the definition caches differently with eps and with eps rounded to 32
    bits (some in a million): both kernels write what the definition says."""
    from realizar_b200 import ops
    d, eps = 64, 1e-5
    ones = torch.ones(d, device="cuda")
    g, found = torch.Generator(device="cuda").manual_seed(1), []
    for _ in range(8):
        x = 1e-3 * torch.randn(1 << 20, 1, d, generator=g, device="cuda")
        a, b = (_quant64(_head64(x, ones, None, None, 0, 0, eps=e)) for e in (eps, float(np.float32(eps))))
        found.append(x[(a != b).any(-1)[:, 0], 0])
    k = torch.cat(found)
    n = k.shape[0]
    assert n >= 8
    want = _quant64(_head64(k[:, None], ones, None, None, 0, 0, eps=eps))
    qkv = torch.cat([torch.randn(n, d, device="cuda"), k, k], -1).contiguous()
    pos, pages = torch.zeros(n, device="cuda", dtype=torch.int32), torch.arange(n, device="cuda", dtype=torch.int32)
    kv = [ops.kv_cache_alloc(1, n, 1, d, "cuda", "q4")[:, 0] for _ in range(2)]
    ops.qk_norm_rope_append(qkv, pos, pages, kv[0][0], kv[0][1], 1, 1, d, q_out=torch.empty(n, d, device="cuda"), q_norm_w=ones, k_norm_w=ones, eps=eps)
    partial, counters = ops.attn_decode_scratch(n, 1, 1, d, "cuda", kv_dtype="q4")
    ops.attn_decode_launch(ops.build_attn_decode_params(qkv, torch.empty(n, d, device="cuda"), kv[1][0], kv[1][1], pos, pages[:, None], partial, counters, 1, 1, d, 1, n,
                                                        0, 0, 1e4, 0, d, 2 * d, ones, ones, eps))
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    for c in kv:
        assert torch.equal(ops.kv_pages_to_float(c[0], d, False)[:, 0, 0], want[:, 0])
    assert torch.equal(kv[0], kv[1])


@pytest.mark.parametrize("name", ["q_norm_w", "k_norm_w", "rope_table", "partial", "counters"])
def test_decode_refuses_tensors_of_another_device(cuda_device, name):
    from realizar_b200 import ops
    kv = ops.kv_cache_alloc(1, 3, 2, 64, "cuda", "q4")
    z = lambda *s: torch.zeros(*s, device="cuda")                                                           # noqa: E731
    partial, counters = ops.attn_decode_scratch(2, 4, 1, 64, "cuda", kv_dtype="q4")
    a = dict(qkv=z(2, 512), out=z(2, 256), k_cache=kv[0, 0], v_cache=kv[1, 0], positions=z(2).int(), page_table=z(2, 2).int(), partial=partial, counters=counters, n_heads=4,
             n_kv_heads=2, head_dim=64, splits=1, batch=2, rope_dim=64, rope_type=0, rope_theta=1e4, q_off=0, k_off=256, v_off=384, q_norm_w=z(64), k_norm_w=z(64),
             rope_table=z(5, 32, 2))
    ops.build_attn_decode_params(**a)
    with pytest.raises(ValueError, match="one device"):
        ops.build_attn_decode_params(**{**a, name: a[name].cpu()})


@pytest.mark.parametrize("how", ["reset", "status"])
def test_engine_leaves_no_arrival_counter_raised(cuda_device, how, monkeypatch):
    """After a failed launch (stood in for by a counter that is not zero, and by the status that is read) the engine's next prompt starts
    from counters of zero."""
    from test_gpu_engine import _kq_llama
    from realizar_b200 import ops
    from realizar_b200.models.weights import synthetic_weights
    from realizar_b200.runtime.engine import DecodeEngine, EngineConfig
    cfg = _kq_llama()
    eng = DecodeEngine(synthetic_weights(cfg, seed=21, std=0.05), EngineConfig(max_batch=2, max_seq_len=160, greedy_only=True, kv_dtype="q4", prefill_chunk=64))
    toks = [int(t) for t in np.random.default_rng(8).integers(0, cfg.vocab_size, 90)]
    eng.open_slot(0, 128)
    first = eng.prefill(0, toks)
    counters = eng.batched().prefill_scratch.view(torch.int32)[:640]
    assert not bool(counters.any())
    counters[::3] = 1
    if how == "reset":
        eng.reset()
    else:
        with monkeypatch.context() as m:
            m.setattr(ops, "device_error", lambda clear=True: 3115)
            with pytest.raises(ops.KernelError, match="3115"):
                eng.check_health()
        eng.close_slot(0)
    assert not bool(counters.any())
    eng.open_slot(0, 128)
    assert eng.prefill(0, toks) == first
    eng.close()


# ------------------------------------------------------------------------------------------------ prompt attention divided evenly over the SMs
class _Divided:
    """A prompt chunk for which the launcher divides the key tiles evenly (few row tiles over many keys: a cluster of eight CTAs to each would
    leave most SMs idle), with a workspace of its own.  ``used`` tells whether parts went through it since the last ``fresh``."""

    def __init__(self, h, kvh, d, rows, pos0, seed=0, window=0, dtype=torch.bfloat16, scales=None):
        from realizar_b200 import ops
        self.ops, self.shape, self.rows, self.pos0, self.window = ops, (h, kvh, d), rows, pos0, window
        g, total = torch.Generator(device="cuda").manual_seed(seed + d), pos0 + rows
        per = -(-total // 16)
        self.kc, self.vc = _cache(per + 2, kvh, d, seed=seed)
        self.pt = torch.randperm(per + 2, generator=g, device="cuda").to(torch.int32)[:per].contiguous()
        if scales is not None:
            sc = scales(torch.arange(16 * per, device="cuda").float())
            for k in range(kvh):
                self.vc.flatten(-2)[self.pt.long(), k, 8 * d:] = torch.stack([sc, -7.5 * sc], -1).bfloat16().view(torch.uint8).view(-1, 64)
        self.qkv = torch.randn(rows, (h + 2 * kvh) * d, generator=g, device="cuda")
        self.out = torch.full((rows, h * d), 9.0, device="cuda", dtype=dtype)
        self.scratch = ops.attn_prefill_scratch(rows, h, kvh, d, "cuda")
        self.fresh()

    def fresh(self):
        self.scratch[640:] = 7.0
        self.out.fill_(9.0)

    def used(self):
        assert not bool(self.scratch[:640].any())                  # the arrival counters are zero again
        return bool((self.scratch[640:] != 7.0).any())

    def launch(self, **kw):
        h, kvh, d = self.shape
        a = dict(window=self.window, scratch=self.scratch, pos0=self.pos0)
        a.update(kw)
        self.ops.attn_prefill(self.qkv, a.pop("out", self.out), self.kc, self.vc, self.pt, self.rows, a.pop("pos0"), h, kvh, d, **a)

    def check(self, out=None, pos0=None):
        torch.cuda.synchronize()
        assert self.ops.device_error() == 0
        h, kvh, d = self.shape
        pos0 = self.pos0 if pos0 is None else pos0
        n, out = pos0 + self.rows, self.out if out is None else out
        ks, vs = _gather(self.kc, self.pt, d, False, n), _gather(self.vc, self.pt, d, True, n)
        worst = 0.0
        for r in range(self.rows):
            p1 = pos0 + r + 1
            want = _attend64(self.qkv[r, : h * d].double().view(h, d), ks[:, :p1], vs[:, :p1], max(0, p1 - self.window) if self.window else 0)
            worst = max(worst, _rel(out[r], want))
        assert worst < 3 * 4e-3, worst                              # (of a single row, as in _prompt)


@pytest.mark.parametrize("h, kvh, d, rows, pos0, kw", [
    (4, 2, 128, 40, 9000, {}), (2, 2, 96, 40, 9000, {}), (14, 2, 64, 40, 9001, {}), (3, 3, 80, 70, 12345, {}), (6, 1, 96, 100, 20000, dict(window=9000)),
    (8, 2, 128, 40, 9000, dict(dtype=torch.float32)), (2, 2, 96, 200, 7777, {})])
@pytest.mark.parametrize("dev_pos", [False, True])
def test_prompt_of_few_rows_divided_evenly(cuda_device, h, kvh, d, rows, pos0, kw, dev_pos):
    c = _Divided(h, kvh, d, rows, pos0, **kw)
    pd = torch.tensor([pos0], device="cuda", dtype=torch.int32) if dev_pos else None
    for _ in range(2):
        c.launch(**(dict(pos0=0, pos0_dev=pd) if dev_pos else {}))
    c.check()
    assert c.used()
    first = c.out.clone()
    c.fresh()
    c.launch(**(dict(pos0=0, pos0_dev=pd) if dev_pos else {}))
    assert torch.equal(c.out, first) and c.used()                  # the same bits from any workspace


@pytest.mark.parametrize("kind", ["constant first", "growing", "shrinking"])
def test_prompt_divided_evenly_with_wide_ranges_of_scales(cuda_device, kind):
    """The parts of a row come with powers of two of their own."""
    c = _Divided(4, 2, 64, 40, 9000, dtype=torch.float32, scales={"constant first": lambda i: torch.where(i < 4000, 0.0, 1e-6), "growing": lambda i: torch.exp2(i / 400 - 20),
                                                                  "shrinking": lambda i: torch.exp2(5 - i / 400)}[kind])
    c.launch()
    c.check()
    assert c.used()


def test_prompt_divided_evenly_only_with_a_workspace_that_is_large_enough(cuda_device):
    from realizar_b200 import ops
    c = _Divided(4, 2, 128, 40, 9000)
    c.launch()
    c.check()
    assert c.used()
    small = torch.zeros(c.scratch.numel() - 4, device="cuda")
    for scratch in (None, small, ops.attn_prefill_scratch(40, 4, 2, 64, "cuda")):
        out = torch.full_like(c.out, 9.0)
        c.launch(scratch=scratch, out=out)
        c.check(out)
        assert scratch is None or not bool(scratch.any())
    larger = torch.zeros(c.scratch.numel() + 1000, device="cuda")
    out = torch.full_like(c.out, 9.0)
    c.launch(scratch=larger, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, c.out) and bool(larger[640:].any()) and not bool(larger[:640].any()) and not bool(larger[c.scratch.numel():].any())


def test_prompts_divided_evenly_on_two_streams_with_their_own_workspaces(cuda_device):
    jobs = [_Divided(4, 2, 128, 40, 9000, seed=1), _Divided(14, 2, 64, 70, 12000, seed=2)]
    want = []
    for c in jobs:
        c.launch()
        c.check()
        assert c.used()
        want.append(c.out.clone())
        c.fresh()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(20):
        for c, s in zip(jobs, streams):
            with torch.cuda.stream(s):
                c.launch()
    torch.cuda.synchronize()
    for c, w in zip(jobs, want):
        assert torch.equal(c.out, w) and c.used()


def test_captured_prompts_divided_evenly_share_a_workspace(cuda_device):
    """Two graphs with one workspace, replayed in turn at several positions; one of the positions leaves hardly any keys to divide."""
    a, b = _Divided(4, 2, 96, 40, 9000, seed=1), _Divided(8, 2, 96, 40, 11000, seed=2)
    b.scratch = a.scratch
    pos = [torch.tensor([c.pos0], device="cuda", dtype=torch.int32) for c in (a, b)]
    graphs = []
    for c, p in zip((a, b), pos):
        c.launch(pos0=0, pos0_dev=p)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            c.launch(pos0=0, pos0_dev=p)
    for back in (0, 1234, 8990):
        for c, p in zip((a, b), pos):
            p.fill_(c.pos0 - back)
            c.fresh()
        for _ in range(3):
            for g in graphs:
                g.replay()
        for c in (a, b):
            c.check(pos0=c.pos0 - back)
        assert a.used()


# ------------------------------------------------------------------------------------------------ engine, decode steps of a batch
@pytest.mark.parametrize("name", ["llama", "phi2"])
def test_engine_batch_step_over_the_4_bit_cache(cuda_device, name):
    """Several sequences of unequal length with an idle slot between them, in one decode step: on the tensor-core path (append, then attention
    without append over per-row page tables) and on the fused one, both against the same sequences fed one at a time.

    The prompts' rows are the same bytes.  The tensor-core path takes bf16 activations and the other int8 ones, some 1% apart, which moves
    one code in thirty of the few new rows by a step of 0.31 sigma: 0.31 x sqrt(0.03) = 5% of such a row, 1 - 0.05^2 / 2 = 0.999 of its cosine.
    Two layers and the activations themselves stay above the 0.99 that the engine's other tests hold the two paths to."""
    from test_gpu_engine import _cos, _kq_llama, small_phi2
    from realizar_b200.models.weights import synthetic_weights
    from realizar_b200.runtime.engine import DecodeEngine, EngineConfig
    cfg = _kq_llama() if name == "llama" else small_phi2()
    w = synthetic_weights(cfg, seed=21, std=0.05, **({} if name == "llama" else {"scheme": "Q4_K_M"}))
    rng = np.random.default_rng(3)
    lens = {0: 40, 1: 17, 3: 90, 4: 3, 5: 64}                     # slot 2 stays idle
    prompts = {s: [int(t) for t in rng.integers(0, cfg.vocab_size, n)] for s, n in lens.items()}
    steps = [{s: int(rng.integers(0, cfg.vocab_size)) for s in lens} for _ in range(3)]
    res = {}
    for how, min_batch in (("tensor core", 4), ("fused", 64), ("alone", 64)):
        eng = DecodeEngine(w, EngineConfig(max_batch=6, max_seq_len=128, greedy_only=True, kv_dtype="q4", prefill_chunk=64, gemm_decode_min_batch=min_batch))
        assert eng._use_batched_step(eng.bucket_for(6)) == (how == "tensor core")
        for s, p in prompts.items():
            eng.open_slot(s, 128)
            eng.prefill(s, p)
        res[how] = []
        for feed in steps:
            row = {}
            for part in [{s: feed[s]} for s in lens] if how == "alone" else [feed]:
                eng.feed(part)
                row.update({s: eng.logits_of_last_step(s).float().cpu().numpy() for s in part})
            res[how].append(row)
        eng.check_health()
        eng.close()
    for how in ("tensor core", "fused"):
        for a, b in zip(res[how], res["alone"]):
            for s in lens:
                assert _cos(a[s], b[s]) > 0.99, (how, s)


@pytest.mark.parametrize("size", [0.0, 1e-20, 1e-32, 1e-38])
def test_prompt_with_tiny_queries_behind_zero_keys(cuda_device, size):
    """Key tiles of zeros and queries near the smallest numbers: all scores are 0 or next to it, and no tile's keys drop out of the mean."""
    from realizar_b200 import ops
    h, kvh, d, n, rows = 4, 2, 64, 700, 90
    kc, vc = _cache(46, kvh, d)
    pt = torch.randperm(46, device="cuda").to(torch.int32)[:44].contiguous()
    kc.flatten(-2)[pt[:20].long(), :, 8 * d:] = 0                    # the first 320 keys; the rows before the last begin in a tile that is masked in part
    qkv = size * torch.randn(rows, (h + 2 * kvh) * d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    ks, vs = _gather(kc, pt, d, False, n), _gather(vc, pt, d, True, n)
    for first in (n - rows, 100):
        out = torch.empty(rows, h * d, device="cuda")
        ops.attn_prefill(qkv, out, kc, vc, pt, rows, first, h, kvh, d)
        for r in range(0, rows, 7):
            p1 = first + r + 1
            assert _rel(out[r], _attend64(qkv[r, : h * d].double().view(h, d), ks[:, :p1], vs[:, :p1], 0)) < 4e-3, (first, r)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5])
def test_windows_beyond_32_bits_hide_nothing(cuda_device, window):
    _prompt(4, 2, 64, 90, 500, window=window)
    _decode(4, 2, 64, [40, 17], seed=1, window=window)()
