"""Refusals of the 4-bit cache's and 4-bit weights' entry points (no GPU: arguments
are checked before any device work, and these calls carry no context)."""
import ctypes

import pytest

import glacier_attn as ga

INVALID, UNSUPPORTED = ga.ERR_INVALID_ARGUMENT, ga.ERR_UNSUPPORTED
MB = 1 << 20
PAGE = 2 * 18 * 2 * 16  # bytes of a page of _cache()


def _said(rc):
    return rc, ga.load().glacier_attn_last_error().decode()


def _cache(**kw):
    f = dict(k_pages=MB, v_pages=2 * MB, page_stride=PAGE, n_pages=9, page_size=16, n_heads_kv=2, head_dim=64,
             io_dtype=ga.IO_BF16)
    b = dict(cu_tokens=3 * MB, kv_lens=4 * MB, page_table=5 * MB, table_stride=7, n_seqs=3, total_tokens=8,
             max_pages=7, max_new=0, max_kv=0)
    for k, v in kw.items():
        (f if k in f else b)[k] = v
    return ga.KvCache(**f), ga.CacheBatch(**b)


def _append(base=1e4, hq=4, k=6 * MB, v=7 * MB, q=8 * MB, q_rot=9 * MB, **kw):
    c, b = _cache(**kw)
    return _said(ga.load().glacier_attn_qcache_append(None, ctypes.byref(c), ctypes.byref(b), k, v, base, hq, q, q_rot))


def _read(k=6 * MB, v=7 * MB, **kw):
    c, b = _cache(**kw)
    return _said(ga.load().glacier_attn_qcache_read(None, ctypes.byref(c), ctypes.byref(b), k, v))


def _forward(hq=4, q=8 * MB, out=9 * MB, lse=10 * MB, **kw):
    c, b = _cache(**kw)
    return _said(ga.load().glacier_attn_qcache_forward(None, ctypes.byref(c), ctypes.byref(b), hq, q, out, lse, None, 0))


@pytest.mark.parametrize("call", [_append, _read, _forward])
@pytest.mark.parametrize("change,code,word", [
    (dict(n_pages=-1), INVALID, "n_pages"), (dict(n_heads_kv=0), INVALID, "head counts"),
    (dict(head_dim=0), INVALID, "head_dim"), (dict(head_dim=100), UNSUPPORTED, "head_dim"),
    (dict(head_dim=264), UNSUPPORTED, "head_dim"), (dict(io_dtype=2), INVALID, "io dtype"),
    (dict(page_size=8), UNSUPPORTED, "page_size"), (dict(page_size=48), UNSUPPORTED, "page_size"),
    (dict(page_size=2048), UNSUPPORTED, "page_size"), (dict(page_stride=PAGE - 16), INVALID, "page_stride"),
    (dict(page_stride=PAGE + 8), UNSUPPORTED, "multiple of 16"), (dict(page_stride=PAGE + 16), INVALID, "ctx"),
    (dict(head_dim=160), INVALID, "page_stride"),  # (six groups, not five)
    (dict(head_dim=160, page_stride=2 * 18 * 6 * 16), INVALID, "ctx"),
    (dict(page_stride=1 << 41), UNSUPPORTED, "too large"), (dict(n_seqs=-1), INVALID, "n_seqs"),
    (dict(total_tokens=-1), INVALID, "total_tokens"), (dict(max_pages=-1), INVALID, "max_pages"),
    (dict(max_new=-1), INVALID, "max_new"), (dict(max_kv=-5), INVALID, "max_kv"),
    (dict(table_stride=6), INVALID, "table_stride"),
    (dict(max_pages=1 << 27, table_stride=1 << 27), UNSUPPORTED, "2^30"),
    (dict(total_tokens=1 << 30), UNSUPPORTED, "too large"), (dict(n_seqs=1 << 21), UNSUPPORTED, "too many sequences"),
    (dict(cu_tokens=None), INVALID, "cu_tokens"), (dict(kv_lens=None), INVALID, "kv_lens"),
    (dict(page_table=None), INVALID, "page_table"), (dict(k_pages=None), INVALID, "k_pages"),
    (dict(v_pages=8), UNSUPPORTED, "v_pages must be 16-byte"), ({}, INVALID, "ctx"),
    (dict(total_tokens=0), INVALID, "ctx"),
    (dict(n_seqs=0, cu_tokens=None, kv_lens=None, page_table=None), INVALID, "ctx"),
    (dict(n_pages=0, k_pages=None, v_pages=None), INVALID, "ctx")])
def test_cache_refusals(call, change, code, word):
    rc, msg = call(**change)
    assert rc == code and word in msg, msg


@pytest.mark.parametrize("change,code,word", [
    (dict(k=None), INVALID, "k is NULL"), (dict(v=6 * MB + 4), UNSUPPORTED, "v must be 16-byte"),
    (dict(base=-2.0), INVALID, "rope_freq_base"), (dict(base=float("nan")), INVALID, "rope_freq_base"),
    (dict(base=0.0), INVALID, "no rotation"), (dict(q_rot=None), INVALID, "q_rot"), (dict(hq=3), INVALID, "multiple"),
    (dict(base=0.0, q=None, q_rot=None, hq=0), INVALID, "ctx"), (dict(q_rot=8 * MB), INVALID, "ctx"),
    (dict(q_rot=8 * MB + 64), INVALID, "q_rot overlaps q"), (dict(q_rot=6 * MB), INVALID, "q_rot overlaps k"),
    (dict(v_pages=MB + PAGE), INVALID, "v_pages overlaps k_pages"), (dict(v_pages=MB), INVALID, "v_pages overlaps"),
    (dict(v_pages=MB + PAGE, page_stride=2 * PAGE), INVALID, "ctx"), (dict(v_pages=MB + 9 * PAGE), INVALID, "ctx"),
    (dict(v_pages=MB + 9 * PAGE - 16), INVALID, "v_pages overlaps"), (dict(k=MB + 16), INVALID, "k overlaps k_pages"),
    (dict(k=MB + 9 * PAGE), INVALID, "ctx"), (dict(q_rot=2 * MB + 8 * PAGE), INVALID, "q_rot overlaps v_pages")])
def test_append_refusals(change, code, word):
    rc, msg = _append(**change)
    assert rc == code and word in msg, msg


@pytest.mark.parametrize("change,code,word", [
    (dict(k=None), INVALID, "k is NULL"), (dict(v=7 * MB + 8), UNSUPPORTED, "v must be 16-byte"),
    (dict(v=6 * MB + 1024), INVALID, "k overlaps v"), (dict(v=6 * MB), INVALID, "overlaps"),
    (dict(k=MB), INVALID, "k overlaps k_pages"), (dict(v=2 * MB + 16), INVALID, "v overlaps v_pages"),
    (dict(v_pages=MB), INVALID, "ctx")])
def test_read_refusals(change, code, word):
    rc, msg = _read(**change)
    assert rc == code and word in msg, msg


@pytest.mark.parametrize("change,code,word", [
    (dict(q=None), INVALID, "q is NULL"), (dict(out=None), INVALID, "out is NULL"), (dict(out=8 * MB), INVALID, "ctx"),
    (dict(out=8 * MB + 16), INVALID, "out overlaps q"), (dict(lse=None), INVALID, "ctx"), (dict(hq=3), INVALID, "multiple"),
    (dict(out=MB), INVALID, "out overlaps k_pages"), (dict(lse=2 * MB + 4), INVALID, "lse overlaps v_pages"),
    (dict(lse=8 * MB), INVALID, "lse overlaps q"), (dict(lse=9 * MB + 64), INVALID, "lse overlaps out"),
    (dict(q=8 * MB + 8), UNSUPPORTED, "q must be 16-byte"), (dict(hq=2 ** 31 - 2), UNSUPPORTED, "too large"),
    (dict(v_pages=MB), INVALID, "ctx")])
def test_forward_refusals(change, code, word):
    rc, msg = _forward(**change)
    assert rc == code and word in msg, msg


def test_null_descriptors_and_sizes():
    L = ga.load()
    c, b = _cache()
    assert _said(L.glacier_attn_qcache_append(None, None, ctypes.byref(b), 16, 16, 0.0, 0, None, None))[0] == INVALID
    assert _said(L.glacier_attn_qcache_read(None, ctypes.byref(c), None, 16, 16))[0] == INVALID
    assert _said(L.glacier_attn_qcache_forward(None, ctypes.byref(c), None, 4, 16, 16, None, None, 0))[0] == INVALID
    assert L.glacier_attn_qcache_workspace(None, ctypes.byref(c), ctypes.byref(b), 4) == 0
    assert L.glacier_attn_qcache_page_bytes(ctypes.byref(c)) == PAGE == 2 * ga.quant_page_bytes(16, 64)
    for d, groups in ((8, 1), (40, 2), (96, 3), (128, 4), (136, 6), (192, 6), (200, 8), (256, 8)):
        wide, _ = _cache(head_dim=d, page_stride=0)
        assert L.glacier_attn_qcache_page_bytes(ctypes.byref(wide)) == 2 * 16 * 18 * groups == 2 * ga.quant_page_bytes(16, d)
    bad, _ = _cache(page_size=24)
    assert L.glacier_attn_qcache_page_bytes(ctypes.byref(bad)) == L.glacier_attn_qcache_page_bytes(None) == 0


# ---- 4-bit weights ----------------------------------------------------------
@pytest.mark.parametrize("out,cols,group,offsets,code,word", [
    (0, 64, 32, 0, INVALID, "out_features"), (16, -32, 32, 0, INVALID, "in_features"),
    (16, 64, 16, 0, UNSUPPORTED, "group"), (16, 64, 0, 0, UNSUPPORTED, "group"), (16, 64, 32, 2, INVALID, "offsets"),
    (18, 64, 32, 0, UNSUPPORTED, "multiple of 4"), (16, 48, 32, 0, UNSUPPORTED, "multiple of 32"),
    (16, 96, 64, 0, UNSUPPORTED, "of group"), (1 << 20, 2048, 32, 0, UNSUPPORTED, "too large"),
    (4, 1 << 24, 32, 0, UNSUPPORTED, "too large"), (4, (1 << 24) - 32, 32, 0, None, "")])
def test_sizes_of_weights(out, cols, group, offsets, code, word):
    L, w = ga.load(), ga.QuantWeights(out, cols, group, offsets)
    size = L.glacier_proj_quant_bytes(ctypes.byref(w))
    if code is None:
        assert size == 16 * cols // 128 * 128 // 2 + 16 * cols // 32 * 2 + 16 * (-cols % 128) * 9 // 16
        return
    assert size == 0
    rc, msg = _said(L.glacier_proj_quant_pack(None, ctypes.byref(w), MB, 2 * MB, 3 * MB if offsets else None, 4 * MB))
    assert rc == code and word in msg, msg
    with pytest.raises(ga.GlacierAttnError):
        ga._packed_bytes(out, cols, group, offsets)


def _pack(numbers=MB, scales=2 * MB, offsets=3 * MB, packed=4 * MB, out=64, cols=256, group=64, has=1):
    w = ga.QuantWeights(out, cols, group, has)
    return _said(ga.load().glacier_proj_quant_pack(None, ctypes.byref(w), numbers, scales, offsets, packed))


@pytest.mark.parametrize("change,code,word", [
    ({}, INVALID, "ctx"), (dict(numbers=None), INVALID, "numbers is NULL"), (dict(scales=None), INVALID, "scales is NULL"),
    (dict(packed=None), INVALID, "packed is NULL"), (dict(offsets=None), INVALID, "offsets is NULL"),
    (dict(has=0), INVALID, "offsets are given"), (dict(packed=4 * MB + 8), UNSUPPORTED, "16-byte"),
    (dict(scales=2 * MB + 1), UNSUPPORTED, "2-byte"), (dict(offsets=3 * MB + 1), UNSUPPORTED, "2-byte"),
    (dict(packed=MB), INVALID, "packed overlaps numbers"), (dict(packed=2 * MB - 32), INVALID, "packed overlaps scales"),
    (dict(packed=3 * MB + 256), INVALID, "packed overlaps offsets"), (dict(numbers=MB + 1), INVALID, "ctx")])
def test_pack_refusals(change, code, word):
    rc, msg = _pack(**change)
    assert rc == code and word in msg, msg


def _proj(T=8, cols=256, group=64, offsets=0, rank=16, io=ga.IO_BF16, x=MB, n=2, work=20 * MB, work_bytes=1 << 30,
          **change):
    L, arr = ga.load(), (ga.LoraProj * max(n, 5))()
    for i in range(len(arr)):
        arr[i] = ((2 + 3 * i) * MB, None, (3 + 3 * i) * MB, (4 + 3 * i) * MB, 1.0, 64, (3 + 3 * i) * MB + MB // 2, None,
                  None, None)
    for k, v in change.items():
        setattr(arr[1], k, v)
    desc = ga.QuantProjDesc(T, cols, group, offsets, rank, io)
    return _said(L.glacier_proj_quant_forward(None, ctypes.byref(desc), x, arr, n, work, work_bytes)), (
        L.glacier_proj_quant_workspace(ctypes.byref(desc), arr, n))


@pytest.mark.parametrize("change,code,word", [
    ({}, INVALID, "ctx"), (dict(T=-1), INVALID, "total_tokens"), (dict(T=0), INVALID, "ctx"),
    (dict(io=4), INVALID, "io dtype"), (dict(n=0), INVALID, "n_proj"), (dict(n=5), INVALID, "n_proj"),
    (dict(group=48), UNSUPPORTED, "group"), (dict(offsets=3), INVALID, "offsets"), (dict(cols=40), UNSUPPORTED, "32"),
    (dict(rank=0), INVALID, "rank"), (dict(rank=65), INVALID, "rank"), (dict(rank=64), INVALID, "ctx"),
    (dict(T=1 << 23), UNSUPPORTED, "too large"), (dict(T=1 << 26, cols=32, group=32), UNSUPPORTED, "too large"),
    (dict(x=None), INVALID, "x is NULL"), (dict(x=MB + 8), UNSUPPORTED, "x must be 16-byte"),
    (dict(w=None), INVALID, "proj[1].w is NULL"), (dict(w=5 * MB + 4), UNSUPPORTED, "proj[1].w must be"),
    (dict(y=None), INVALID, "proj[1].y is NULL"), (dict(y=6 * MB + 8), UNSUPPORTED, "proj[1].y must be"),
    (dict(lora_a=6 * MB + 4), UNSUPPORTED, "lora_a must be"), (dict(lora_b=None), INVALID, "lora_b is NULL"),
    (dict(lora_b=7 * MB + 4), UNSUPPORTED, "lora_b must be"), (dict(scaling=float("inf")), INVALID, "scaling"),
    (dict(out_features=0), INVALID, "out_features"), (dict(out_features=66), UNSUPPORTED, "multiple of 4"),
    (dict(out_features=1 << 24), UNSUPPORTED, "too large"),
    (dict(lora_a=None, lora_b=None, rank=0), INVALID, "rank"),  # (the other projection has one)
    (dict(y=MB + 16), INVALID, "proj[1].y overlaps x"), (dict(y=2 * MB), INVALID, "proj[1].y overlaps proj[0].w"),
    (dict(y=5 * MB + 64), INVALID, "proj[1].y overlaps proj[1].w"), (dict(y=3 * MB), INVALID, "overlaps proj[0].lora_a"),
    (dict(y=4 * MB), INVALID, "overlaps proj[0].lora_b"), (dict(y=3 * MB + MB // 2), INVALID, "overlaps proj"),
    (dict(bias=6 * MB + MB // 2), INVALID, "overlaps proj[1].bias"), (dict(bias=9 * MB), INVALID, "ctx"),
    (dict(work=None), INVALID, "workspace is NULL"), (dict(work=20 * MB + 16), INVALID, "256-byte"),
    (dict(work_bytes=64), INVALID, "workspace of 64 bytes")])
def test_product_refusals(change, code, word):
    (rc, msg), _ = _proj(**change)
    assert rc == code and word in msg, msg


def test_product_workspace():
    L = ga.load()
    _, both = _proj()
    _, one = _proj(lora_a=None)
    assert both == 2 * one > 0
    for kw in ({}, dict(T=40), dict(T=40, io=ga.IO_F32), dict(io=ga.IO_F32)):
        _, size = _proj(**kw)
        assert _proj(work_bytes=size, **kw)[0][1].startswith("ctx")
        assert "workspace" in _proj(work_bytes=size - 1, **kw)[0][1]
    plain = (ga.LoraProj * 1)((MB, None, None, None, 0.0, 64, 2 * MB, None, None, None))
    for io, size in ((ga.IO_BF16, 0), (ga.IO_F32, 3 * 2 * 8 * 256)):
        desc = ga.QuantProjDesc(8, 256, 64, 0, 0, io)
        assert L.glacier_proj_quant_workspace(ctypes.byref(desc), plain, 1) == size
    assert L.glacier_proj_quant_workspace(None, plain, 1) == L.glacier_proj_quant_workspace(ctypes.byref(desc), None, 1) == 0
    assert _said(L.glacier_proj_quant_forward(None, None, MB, plain, 1, None, 0))[0] == INVALID
    assert _said(L.glacier_proj_quant_forward(None, ctypes.byref(desc), MB, None, 1, None, 0))[0] == INVALID


# ---- the front end ----------------------------------------------------------
def _good():
    torch = pytest.importorskip("torch")
    kp = torch.zeros(4, 2, ga.quant_page_bytes(16, 64), dtype=torch.uint8)
    return torch, dict(k_pages=kp, v_pages=kp.clone(), cu_tokens=torch.zeros(2, dtype=torch.int32),
                       kv_lens=torch.zeros(1, dtype=torch.int32), page_table=torch.zeros(1, 3, dtype=torch.int32),
                       total_tokens=1, max_new=0, max_kv=0, device=-1,  # -1: the device of CPU tensors
                       head_dim=64, dtype=torch.bfloat16)


def test_front_end_checks_tensors_before_the_abi():
    torch, good = _good()
    kp = good["k_pages"]
    cache, batch = ga.qcache_args(**good)
    assert (cache.page_stride, cache.n_pages, cache.page_size, cache.head_dim) == (PAGE, 4, 16, 64)
    assert cache.io_dtype == ga.IO_BF16 and (batch.n_seqs, batch.max_pages, batch.table_stride) == (1, 3, 3)
    both = torch.zeros(4, 2, 2, ga.quant_page_bytes(16, 64), dtype=torch.uint8)
    cache, _ = ga.qcache_args(**dict(good, k_pages=both[:, 0], v_pages=both[:, 1], dtype=torch.float32))
    assert cache.page_stride == 2 * PAGE and cache.v_pages - cache.k_pages == PAGE and cache.io_dtype == ga.IO_F32
    for change in (dict(k_pages=kp[0]), dict(v_pages=kp.float()), dict(v_pages=kp[:3]), dict(v_pages=both[:, 1]),
                   dict(k_pages=kp.to(torch.int8), v_pages=kp.to(torch.int8)), dict(head_dim=0), dict(head_dim=-4),
                   dict(k_pages=kp[:, :, ::2], v_pages=kp[:, :, ::2]), dict(k_pages=kp[:, :, :-4], v_pages=kp[:, :, :-4]),
                   dict(dtype=torch.float16), dict(kv_lens=good["cu_tokens"]), dict(cu_tokens=good["cu_tokens"].long()),
                   dict(page_table=good["page_table"][0]), dict(device=0)):
        with pytest.raises(TypeError):
            ga.qcache_args(**dict(good, **change))
    # (a page's size is what its bytes say: of another head size it may not be one that is taken)
    cache, _ = ga.qcache_args(**dict(good, head_dim=128))
    assert cache.page_size == 8


def test_sizes_past_32_bits_are_refused_not_wrapped():
    torch, good = _good()
    big = 2 ** 32 + 5
    pages = torch.empty(big, 2, ga.quant_page_bytes(16, 64), dtype=torch.uint8, device="meta")
    for change in (dict(total_tokens=big), dict(k_pages=pages, v_pages=pages),
                   dict(page_table=torch.empty(1, big, dtype=torch.int32, device="meta")), dict(head_dim=2 ** 40)):
        with pytest.raises((ga.Unsupported, TypeError)):
            ga.qcache_args(**dict(good, **change))
    for sizes in ((big, 64, 32, 0), (64, 2 ** 32 + 64, 32, 0), (64, 64, big, 0)):
        with pytest.raises(ga.Unsupported, match="too large"):
            ga._packed_bytes(*sizes)
        with pytest.raises(ga.Unsupported, match="too large"):
            ga.GpuAttentionEngine.quant_bytes(*sizes)


def test_front_end_checks_products():
    torch = pytest.importorskip("torch")
    import types

    eng = types.SimpleNamespace(device_ordinal=-1, _io_of=ga.GpuAttentionEngine._io_of)
    forward, pack = ga.GpuAttentionEngine.proj_quant_forward, ga.GpuAttentionEngine.quant_pack
    x, size = torch.zeros(3, 64), ga._packed_bytes(8, 64, 32, 0)
    good = dict(w=torch.zeros(size, dtype=torch.uint8), out=8, a=torch.zeros(64, 4), b=torch.zeros(4, 8))
    for bad in (dict(w=good["w"][:-1]), dict(w=good["w"].to(torch.int8)), dict(a=torch.zeros(64, 5)),
                dict(b=torch.zeros(8, 4)), dict(b=torch.zeros(4, 8, dtype=torch.bfloat16)), dict(bias=torch.zeros(9)),
                dict(y=torch.zeros(3, 9)), dict(y=torch.zeros(3, 8, dtype=torch.bfloat16)),
                dict(y=torch.zeros(8, 3).t())):
        with pytest.raises(TypeError):
            forward(eng, x, [dict(good, **bad)], rank=4)
    for wrong in (x[0], x.half(), x[:, ::2]):
        with pytest.raises((TypeError, ga.Unsupported)):
            forward(eng, wrong, [good], rank=4)
    with pytest.raises(ga.Unsupported):
        forward(eng, x, [dict(good, out=10)], rank=4)
    n, s = torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 2, dtype=torch.float16)
    for args in ((n[0], s), (n, s[0]), (n, s[:, :0]), (n.to(torch.int8), s), (n, s.float()), (n, s[:4]),
                 (n, s, s[:, :1]), (n, s, None, torch.zeros(size - 1, dtype=torch.uint8))):
        with pytest.raises((TypeError, ga.Unsupported)):
            pack(types.SimpleNamespace(device_ordinal=-1), *args)


def test_a_projection_is_written_at_once():
    arr = (ga.LoraProj * 2)()
    ga._LORA_PROJ.pack_into(arr, ga._LORA_PROJ.size, 1, 2, 3, 4, -1.5, 6, 7, 8, 9, 10)
    assert ga._LORA_PROJ.size == ctypes.sizeof(ga.LoraProj) and not arr[0].w
    assert [getattr(arr[1], f) for f, _ in ga.LoraProj._fields_] == [1, 2, 3, 4, -1.5, 6, 7, 8, 9, 10]


def test_rows_to_be_quantised():
    torch = pytest.importorskip("torch")
    for w, group in ((torch.zeros(4, 40), 32), (torch.zeros(32), 32), (torch.zeros(4, 64), 0), (torch.zeros(4, 64), 128)):
        with pytest.raises(TypeError):
            ga.quantise_rows(w, group)
    numbers, scales = ga.quantise_rows(torch.tensor([[0.0, -4.0, 4.0, 1.0]]).repeat(4, 16), 32)
    assert (scales == -0.5).all() and (numbers[:, 0] == (8 | 15 << 4)).all() and (numbers[:, 1] == (0 | 6 << 4)).all()
    numbers, scales = ga.quantise_rows(torch.zeros(4, 64), 64)
    assert not scales.any() and (numbers == 0x88).all()
