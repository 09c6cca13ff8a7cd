"""4-bit KV cache: page layout and refusals of the entry points (no GPU needed)."""
import pytest
import torch

from realizar_b200 import ops


@pytest.mark.parametrize("d", ops.Q4_HEAD_DIMS)
@pytest.mark.parametrize("values", [False, True])
def test_page_layout_is_a_bijection_and_decodes(d, values):
    """Every byte of the code area holds one (token, pair of dims); decoding a page built through that table returns what went in."""
    at = ops._q4_byte_order(d, values, "cpu")
    assert sorted(at.flatten().tolist()) == list(range(8 * d))
    g = torch.Generator().manual_seed(d)
    code = torch.randint(0, 16, (3, 2, 16, d), generator=g, dtype=torch.uint8)
    meta = torch.randn(3, 2, 16, 2, generator=g).bfloat16()
    page = torch.zeros(3, 2, 16 * (d // 2 + 4), dtype=torch.uint8)
    page[..., at.flatten()] = (code[..., 0::2] | code[..., 1::2] << 4).flatten(-2)
    page[..., 8 * d:] = meta.view(torch.uint8).flatten(-2)
    got = ops.kv_pages_to_float(page.view(3, 2, 16, d // 2 + 4), d, values)
    assert torch.equal(got, code.float() * meta[..., :1].float() + meta[..., 1:].float())


def test_cache_formats_and_sizes():
    kv = ops.kv_cache_alloc(2, 5, 3, 80, "cpu", "q4")
    assert kv.shape == (2, 2, 5, 3, 16, 44) and kv.dtype == torch.uint8
    assert [ops.kv_format(ops.kv_cache_alloc(1, 2, 1, 64, "cpu", t), 64) for t in ("bf16", "q8", "q4")] == [ops.KV_BF16, ops.KV_Q8, ops.KV_Q4]
    assert [ops.kv_row_bytes(128, t) for t in ("bf16", "q8", "q4")] == [256, 144, 68]
    q8 = ops.kv_cache_alloc(1, 2, 1, 64, "cpu", "q8")[0, 0]
    assert torch.equal(ops.kv_pages_to_float(q8, 64, True), ops.kv_rows_to_float(q8, 64))
    for bad in (dict(head_dim=72), dict(head_dim=256), dict(head_dim=64, page=32)):
        with pytest.raises(ValueError):
            ops.kv_cache_alloc(1, 2, 1, device="cpu", dtype="q4", **bad)
    with pytest.raises(ValueError):
        ops.kv_cache_alloc(1, 2, 1, 64, "cpu", "q3")
    with pytest.raises(ValueError):
        ops.kv_row_bytes(64, "q3")
    with pytest.raises(ValueError):
        ops.kv_rows_to_float(kv[0, 0], 80)


def _append_args(d=64, n=4, h=4, kvh=2):
    kv = ops.kv_cache_alloc(1, 3, kvh, d, "cpu", "q4")
    return dict(qkv=torch.zeros(n, (h + 2 * kvh) * d), positions=torch.zeros(n, dtype=torch.int32), page_rows=torch.zeros(n, dtype=torch.int32),
                k_cache=kv[0, 0], v_cache=kv[1, 0], n_heads=h, n_kv_heads=kvh, head_dim=d)


@pytest.mark.parametrize("change, word", [
    (dict(qkv=torch.zeros(4, 100)), "qkv"), (dict(qkv=torch.zeros(4, 512).half()), "qkv"), (dict(qkv=torch.zeros(512, 4).t()), "qkv"),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), "positions"), (dict(positions=torch.zeros(4, dtype=torch.int64)), "positions"),
    (dict(page_rows=torch.zeros(8, dtype=torch.int32)[::2]), "page_rows"), (dict(qkv=torch.zeros(4, 513)[:, 1:]), "8-byte"), (dict(q_out=torch.zeros(4, 257)[:, :256]), "8-byte"), (dict(q_out=torch.zeros(4, 100)), "q_out"), (dict(q_out=torch.zeros(3, 256)), "q_out"),
    (dict(q_norm_w=torch.ones(64)), "together"), (dict(q_norm_w=torch.ones(64), k_norm_w=torch.ones(32)), "norm weights"),
    (dict(rope_dim=33), "rope_dim"), (dict(rope_dim=66), "rope_dim"), (dict(rope_dim=-2), "rope_dim"),
    (dict(rope_dim=64, rope_table=torch.zeros(5, 16, 2)), "rope_table"), (dict(n_heads=3), "divide"), (dict(head_dim=48), "4-bit"), (dict(n_kv_heads=4, n_heads=4), "4-bit cache is"),
    (dict(k_cache=torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)), "4-bit"), (dict(v_cache=torch.zeros(2, 2, 16, 36, dtype=torch.uint8)), "differ"),
    (dict(v_cache=torch.zeros(3, 2, 16, 72, dtype=torch.uint8)[..., ::2]), "contiguous"), ({}, "current CUDA device")])
def test_append_refuses(change, word):
    with pytest.raises(ValueError, match=word):
        ops.qk_norm_rope_append(**{**_append_args(), **change})


def test_other_entry_points_refuse_4_bit_caches_they_cannot_serve():
    a = _append_args()
    with pytest.raises(ValueError, match="qk_norm_rope_append"):
        ops.kv_append(a["qkv"][:, 256:], a["qkv"][:, 384:], a["k_cache"], a["v_cache"], a["positions"], a["page_rows"], 2, 64)


def _decode_args(d=64, b=2, h=4, kvh=2):
    kv = ops.kv_cache_alloc(1, 3, kvh, d, "cpu", "q4")
    return dict(qkv=torch.zeros(b, (h + 2 * kvh) * d), out=torch.zeros(b, h * d), k_cache=kv[0, 0], v_cache=kv[1, 0], positions=torch.zeros(b, dtype=torch.int32),
                page_table=torch.zeros(b, 2, dtype=torch.int32), partial=torch.zeros(10), counters=torch.zeros(b * h, dtype=torch.int32), n_heads=h, n_kv_heads=kvh,
                head_dim=d, splits=1, batch=b, rope_dim=0, rope_type=0, rope_theta=1e4, q_off=0, k_off=h * d, v_off=(h + kvh) * d)


@pytest.mark.parametrize("change, word", [
    (dict(batch=0), "batch"), (dict(batch=3), "batch"), (dict(counters=torch.zeros(7, dtype=torch.int32)), "batch"), (dict(page_table=torch.zeros(1, 2, dtype=torch.int32)), "page_table"),
    (dict(out=torch.zeros(2, 256).bfloat16()), "float32"), (dict(positions=torch.zeros(2, dtype=torch.int64)), "int32"), (dict(q_norm_w=torch.ones(64)), "together"),
    (dict(v_cache=torch.zeros(3, 2, 16, 72, dtype=torch.uint8)), "4-bit"), ({}, "current CUDA device")])
def test_decode_refuses(change, word):
    with pytest.raises(ValueError, match=word):
        ops.build_attn_decode_params(**{**_decode_args(), **change})


@pytest.mark.parametrize("change, word", [
    (dict(qkv=torch.zeros(2, 511)), "qkv"), (dict(qkv=torch.zeros(2, 384)), "qkv"), (dict(q_off=-64), "qkv"), (dict(q_off=320), "qkv"), (dict(k_off=448), "qkv"),
    (dict(v_off=448), "qkv"), (dict(v_off=-1), "qkv"), (dict(q_off=320, no_append=True), "qkv"), (dict(qkv=torch.zeros(1024)), "qkv"), (dict(ld_qkv=256), "qkv"),
    (dict(out=torch.zeros(2, 255)), "out"), (dict(out=torch.zeros(512)), "out"), (dict(ld_out=512), "out"), (dict(out=torch.zeros(1, 256).expand(2, 256)), "overlap"),
    (dict(out=torch.zeros(512).as_strided((2, 256), (192, 1))), "overlap"),
    (dict(page_table=torch.zeros(4, dtype=torch.int32)), "page_table"), (dict(page_table=torch.zeros(2, 2, 2, dtype=torch.int32)), "page_table"),
    (dict(q_norm_w=torch.ones(64), k_norm_w=torch.ones(32)), "norm weights"), (dict(q_norm_w=torch.ones(64).half(), k_norm_w=torch.ones(64)), "norm weights"),
    (dict(q_norm_w=torch.ones(128)[::2], k_norm_w=torch.ones(64)), "norm weights"), (dict(rope_dim=64, rope_table=torch.zeros(5, 16, 2)), "rope_table"),
    (dict(rope_dim=64, rope_table=torch.zeros(5, 32, 2).half()), "rope_table"), (dict(rope_dim=33), "rope_dim"), (dict(rope_dim=66), "rope_dim"), (dict(window=-1), "window"),
    (dict(partial=torch.zeros(10).half()), "partial"), (dict(partial=torch.zeros(20)[::2]), "partial"), (dict(counters=torch.zeros(8)), "counters"),
    (dict(counters=torch.zeros(16, dtype=torch.int32)[::2]), "counters"), (dict(n_heads=3), "divide"), (dict(n_heads=0), "divide")])
def test_decode_refuses_what_append_and_prompt_refuse(change, word):
    """What would be read or written out of range, or read as another type."""
    with pytest.raises(ValueError, match=word):
        ops.build_attn_decode_params(**{**_decode_args(), **change})


def test_decode_refuses_rows_that_append_to_one_sequence():
    """Rows of one sequence would read each other's new rows while they are written."""
    with pytest.raises(ValueError, match="no_append"):
        ops.build_attn_decode_params(**{**_decode_args(), "page_table": torch.zeros(4, dtype=torch.int32), "shared_table": True})


@pytest.mark.parametrize("change", [dict(no_append=True, k_off=0, v_off=0, qkv=torch.zeros(2, 256)), dict(page_table=torch.zeros(4, dtype=torch.int32), shared_table=True, no_append=True),
                                    dict(page_table=torch.zeros(4, dtype=torch.int32), shared_table=True, batch=1), dict(page_table=torch.zeros(4, dtype=torch.int32), batch=1),
                                    dict(qkv=torch.zeros(2, 600)[:, 8:], out=torch.zeros(2, 300)[:, 4:]), dict(batch=1, ld_qkv=7, ld_out=7)])
def test_decode_takes_calls_that_are_in_order(change):
    """(up to the check of the device, which is the last but one)"""
    with pytest.raises(ValueError, match="current CUDA device"):
        ops.build_attn_decode_params(**{**_decode_args(), **change})


@pytest.mark.parametrize("change, word", [
    (dict(n_tokens=0), "n_tokens"), (dict(n_tokens=5), "qkv"), (dict(pos0=29), "not covered"), (dict(pos0=-1), "not covered"), (dict(out=torch.zeros(4, 100)), "out"),
    (dict(out=torch.zeros(4, 256).half()), "out"), (dict(page_table=torch.zeros(2, 2, dtype=torch.int32)), "page_table"), (dict(window=-1), "covered"),
    (dict(scratch=torch.zeros(4, dtype=torch.int32)), "scratch"), (dict(pos0_dev=torch.zeros(1)), "pos0_dev"), ({}, "current CUDA device")])
def test_prefill_refuses(change, word):
    kv = ops.kv_cache_alloc(1, 3, 2, 64, "cpu", "q4")
    a = dict(qkv=torch.zeros(4, 512), out=torch.zeros(4, 256), k_cache=kv[0, 0], v_cache=kv[1, 0], page_table=torch.zeros(2, dtype=torch.int32), n_tokens=4, pos0=0,
             n_heads=4, n_kv_heads=2, head_dim=64)
    with pytest.raises(ValueError, match=word):
        ops.attn_prefill(**{**a, **change})


@pytest.mark.parametrize("change, word", [
    (dict(out=torch.zeros(4, 258)[:, 2:]), "16-byte"), (dict(out=torch.zeros(4, 259)[:, :256]), "16-byte"), (dict(out=torch.zeros(1, 256).expand(4, 256)), "overlap"),
    (dict(impl="mma"), "mma"), (dict(n_heads=3), "divide"), (dict(q_off=-64), "qkv"), (dict(page_table=torch.zeros(4, dtype=torch.int32)[::2]), "page_table")])
def test_prefill_refuses_layouts(change, word):
    kv = ops.kv_cache_alloc(1, 3, 2, 64, "cpu", "q4")
    a = dict(qkv=torch.zeros(4, 512), out=torch.zeros(4, 256), k_cache=kv[0, 0], v_cache=kv[1, 0], page_table=torch.zeros(2, dtype=torch.int32), n_tokens=4, pos0=0,
             n_heads=4, n_kv_heads=2, head_dim=64)
    with pytest.raises(ValueError, match=word):
        ops.attn_prefill(**{**a, **change})


def test_append_refuses_overlapping_results():
    with pytest.raises(ValueError, match="overlap"):
        ops.qk_norm_rope_append(**_append_args(), q_out=torch.zeros(1, 256).expand(4, 256))


def test_cli_offers_the_format():
    from realizar_b200.cli import build_parser
    assert build_parser().parse_args(["run", "m.gguf", "hi", "--kv-dtype", "q4"]).kv_dtype == "q4"


def test_append_parameters_are_packed_as_the_structure_lies():
    import ctypes
    from realizar_b200.ops import _signatures as S
    values = [11 * (i + 1) for i in range(11)] + [1e-6] + list(range(1, 9)) + [5e5, 0]
    assert bytes(S.QkAppendParams(*values)) == S.pack_qk_append(*values)
    assert len(S.pack_qk_append(*values)) == ctypes.sizeof(S.QkAppendParams)


def test_library_handle_is_published_with_its_signatures(monkeypatch):
    """Another thread that asks for the kernel library while its signatures are being declared waits for them: calls through an undeclared
    function would pass pointers as 32-bit integers."""
    import threading
    from realizar_b200 import _native
    from realizar_b200.ops import _signatures
    if not _native.cuda_lib_path().exists():
        pytest.skip("kernel library not built")
    declared, entered, seen = threading.Event(), threading.Event(), []
    declare = _signatures.declare

    def slow(lib):
        entered.set()
        second.join(0.3)                                             # time enough to take the handle, if it is there to be taken
        declare(lib)
        declared.set()

    def other():
        entered.wait(10)
        _native.cuda_lib()
        seen.append(declared.is_set())
    monkeypatch.setattr(_native, "_cuda", None)
    monkeypatch.setattr(_signatures, "declare", slow)
    second = threading.Thread(target=other)
    second.start()
    _native.cuda_lib()
    second.join(10)
    assert seen == [True]


@pytest.mark.skipif(torch.cuda.is_available(), reason="other tests may have launched the kernels")
def test_status_of_kernels_that_never_ran_is_not_fetched():
    """Each status word is a synchronous copy from the device (12 us) after every prompt pass: programs without a 4-bit cache do not pay for
    those of its kernels.  (Without a device a copy would answer -1.)"""
    from realizar_b200 import _native
    if not _native.cuda_lib_path().exists():
        pytest.skip("kernel library not built")
    lib = ops.lib()
    assert [lib.rlz_q4_append_error(1), lib.rlz_attn_q4_error(1), lib.rlz_attn_prefill_q4_error(1)] == [0, 0, 0]
