"""Refusals of the q/k norm and paged cache entry points (no GPU: arguments
are checked before any device work, and these calls carry no context)."""
import ctypes

import pytest

import glacier_attn as ga

INVALID, UNSUPPORTED = ga.ERR_INVALID_ARGUMENT, ga.ERR_UNSUPPORTED
MB = 1 << 20


def _said(rc):
    return rc, ga.load().glacier_attn_last_error().decode()


def _norm(T=8, hq=4, hkv=2, d=64, io=ga.IO_BF16, eps=1e-6, base=1e4, backward=False, at=None, work=MB,
          work_bytes=1 << 30):
    L, desc = ga.load(), ga.QkNormDesc(T, hq, hkv, d, io, eps, base)
    # any address: validation fails before it is used
    names = (["dq_out", "dk_out"] if backward else []) + ["q", "k", "q_weight", "k_weight", "positions"] + (
        ["dq", "dk", "dq_weight", "dk_weight"] if backward else ["q_out", "k_out"])
    where = {n: MB * (i + 1) for i, n in enumerate(names)}
    where.update(at or {})
    args = [where[n] for n in names]
    if backward:
        return _said(L.glacier_rmsnorm_qk_backward(None, ctypes.byref(desc), *args, work, work_bytes))
    return _said(L.glacier_rmsnorm_qk_forward(None, ctypes.byref(desc), *args))


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("change,code,word", [
    (dict(T=-1), INVALID, "total_tokens"), (dict(hq=0), INVALID, "head counts"),
    (dict(hkv=-2), INVALID, "head counts"), (dict(d=0), INVALID, "head_dim"),
    (dict(d=60), UNSUPPORTED, "head_dim"), (dict(d=264), UNSUPPORTED, "head_dim"),
    (dict(io=5), INVALID, "io dtype"), (dict(eps=-1.0), INVALID, "eps"),
    (dict(eps=float("nan")), INVALID, "eps"), (dict(base=-1.0), INVALID, "rope_freq_base"),
    (dict(base=float("inf")), INVALID, "rope_freq_base"), (dict(base=float("nan")), INVALID, "rope_freq_base"),
    (dict(T=1 << 29), UNSUPPORTED, "too large"), (dict(at={"q": None}), INVALID, "q is NULL"),
    (dict(at={"k": 24}), UNSUPPORTED, "k must be 16-byte"),
    (dict(at={"k_weight": None}), INVALID, "k_weight"), ({}, INVALID, "ctx"), (dict(T=0), INVALID, "ctx"),
    (dict(base=0.0), INVALID, "ctx"), (dict(at={"positions": None}), INVALID, "ctx"),
    (dict(d=8), INVALID, "ctx"), (dict(d=256), INVALID, "ctx")])
def test_qk_norm_refusals(backward, change, code, word):
    rc, msg = _norm(backward=backward, **change)
    assert rc == code and word in msg, msg


@pytest.mark.parametrize("backward,at,word", [
    (False, {"q_out": MB}, "ctx"), (False, {"k_out": 2 * MB}, "ctx"),
    (False, {"q_out": MB + 16}, "q_out overlaps q"), (False, {"k_out": MB}, "k_out overlaps q"),
    (False, {"q_out": 2 * MB}, "q_out overlaps k"), (False, {"k_out": 6 * MB}, "k_out overlaps q_out"),
    (True, {"dq": MB}, "ctx"), (True, {"dk": 2 * MB}, "ctx"), (True, {"dq": 3 * MB}, "dq overlaps q"),
    (True, {"dk": 4 * MB + 32}, "dk overlaps k"), (True, {"dk": MB}, "dk overlaps dq_out"),
    (True, {"dk_weight": 10 * MB}, "same array"), (True, {"dq_weight": None, "dk_weight": None}, "ctx")])
def test_qk_norm_shared_memory(backward, at, word):
    rc, msg = _norm(backward=backward, at=at)
    assert rc == INVALID and word in msg, msg


def test_qk_norm_workspace():
    need = ga.load().glacier_rmsnorm_qk_workspace(ctypes.byref(ga.QkNormDesc(8, 4, 2, 64, 1, 1e-6, 0.0)))
    assert need > 0
    assert ga.load().glacier_rmsnorm_qk_workspace(ctypes.byref(ga.QkNormDesc(8, 4, 2, 60, 1, 1e-6, 0.0))) == 0
    for kw, word in ((dict(work_bytes=need - 1), "workspace"), (dict(work=None), "workspace"),
                     (dict(work=MB + 16), "256-byte"), (dict(work_bytes=need), "ctx"),
                     (dict(work=None, at={"dq_weight": None, "dk_weight": None}), "ctx")):
        rc, msg = _norm(backward=True, **kw)
        assert rc == INVALID and word in msg, msg


def _cache(**kw):
    f = dict(k_pages=MB, v_pages=2 * MB, page_stride=2 * 16 * 64, n_pages=9, page_size=16, n_heads_kv=2,
             head_dim=64, io_dtype=ga.IO_BF16)
    b = dict(cu_tokens=3 * MB, kv_lens=4 * MB, page_table=5 * MB, table_stride=7, n_seqs=3, total_tokens=8,
             max_pages=7, max_new=0, max_kv=0)
    for k, v in kw.items():
        (f if k in f else b)[k] = v
    return ga.KvCache(**f), ga.CacheBatch(**b)


def _append(base=1e4, hq=4, k=6 * MB, v=7 * MB, q=8 * MB, q_rot=9 * MB, **kw):
    c, b = _cache(**kw)
    return _said(ga.load().glacier_attn_cache_append(None, ctypes.byref(c), ctypes.byref(b), k, v, base, hq, q,
                                                     q_rot))


def _forward(hq=4, q=8 * MB, out=9 * MB, lse=10 * MB, **kw):
    c, b = _cache(**kw)
    return _said(ga.load().glacier_attn_cache_forward(None, ctypes.byref(c), ctypes.byref(b), hq, q, out, lse,
                                                      None, 0))


@pytest.mark.parametrize("call", [_append, _forward])
@pytest.mark.parametrize("change,code,word", [
    (dict(n_pages=-1), INVALID, "n_pages"), (dict(n_heads_kv=0), INVALID, "head counts"),
    (dict(head_dim=0), INVALID, "head_dim"), (dict(head_dim=100), UNSUPPORTED, "head_dim"),
    (dict(head_dim=512), UNSUPPORTED, "head_dim"), (dict(io_dtype=2), INVALID, "io dtype"),
    (dict(page_size=0), UNSUPPORTED, "page_size"), (dict(page_size=8), UNSUPPORTED, "page_size"),
    (dict(page_size=48), UNSUPPORTED, "page_size"), (dict(page_size=2048), UNSUPPORTED, "page_size"),
    (dict(page_stride=2 * 16 * 64 - 8), INVALID, "page_stride"),
    (dict(page_stride=2 * 16 * 64 + 4), UNSUPPORTED, "page_stride"),
    (dict(page_stride=1 << 41), UNSUPPORTED, "too large"), (dict(n_seqs=-1), INVALID, "n_seqs"),
    (dict(total_tokens=-1), INVALID, "total_tokens"), (dict(max_pages=-1), INVALID, "max_pages"),
    (dict(max_new=-1), INVALID, "max_new"), (dict(max_kv=-5), INVALID, "max_kv"),
    (dict(table_stride=6), INVALID, "table_stride"),
    (dict(max_pages=1 << 27, table_stride=1 << 27), UNSUPPORTED, "2^30"),
    (dict(total_tokens=1 << 30), UNSUPPORTED, "too large"), (dict(hq=3), INVALID, "multiple"),
    (dict(hq=0), INVALID, "head counts"), (dict(cu_tokens=None), INVALID, "cu_tokens"),
    (dict(kv_lens=None), INVALID, "kv_lens"), (dict(page_table=None), INVALID, "page_table"),
    (dict(k_pages=None), INVALID, "k_pages"), (dict(v_pages=8), UNSUPPORTED, "v_pages must be 16-byte"),
    (dict(q=8 * MB + 8), UNSUPPORTED, "q must be 16-byte"), ({}, INVALID, "ctx"),
    (dict(n_seqs=0, cu_tokens=None, kv_lens=None, page_table=None), INVALID, "ctx"),
    (dict(n_pages=0, k_pages=None, v_pages=None), INVALID, "ctx"),
    (dict(n_seqs=1, table_stride=0), INVALID, "ctx"), (dict(max_kv=10 ** 9), INVALID, "ctx")])
def test_cache_refusals(call, change, code, word):
    rc, msg = call(**change)
    assert rc == code and word in msg, msg


@pytest.mark.parametrize("change,code,word", [
    (dict(k=None), INVALID, "k is NULL"), (dict(v=None), INVALID, "v is NULL"),
    (dict(k=6 * MB + 4), UNSUPPORTED, "k must be"), (dict(base=-2.0), INVALID, "rope_freq_base"),
    (dict(base=0.0), INVALID, "no rotation"), (dict(q_rot=None), INVALID, "q_rot"),
    (dict(base=0.0, q=None, q_rot=None, hq=0), INVALID, "ctx"), (dict(q=None, q_rot=None), INVALID, "ctx"),
    (dict(q_rot=8 * MB), INVALID, "ctx"), (dict(q_rot=8 * MB + 64), INVALID, "q_rot overlaps q"),
    (dict(q_rot=6 * MB), INVALID, "q_rot overlaps k"), (dict(q_rot=7 * MB + 16), INVALID, "q_rot overlaps v")])
def test_append_refusals(change, code, word):
    rc, msg = _append(**change)
    assert rc == code and word in msg, msg


@pytest.mark.parametrize("change,word", [
    (dict(q=None), "q is NULL"), (dict(out=None), "out is NULL"), (dict(out=8 * MB), "ctx"),
    (dict(out=8 * MB + 16), "out overlaps q"), (dict(lse=None), "ctx")])
def test_forward_refusals(change, word):
    rc, msg = _forward(**change)
    assert rc == INVALID and word in msg, msg


def test_null_descriptors():
    L = ga.load()
    c, b = _cache()
    assert _said(L.glacier_attn_cache_append(None, None, ctypes.byref(b), 16, 16, 0.0, 0, None, None))[0] == INVALID
    assert _said(L.glacier_attn_cache_forward(None, ctypes.byref(c), None, 4, 16, 16, None, None, 0))[0] == INVALID
    assert _said(L.glacier_rmsnorm_qk_forward(None, None, *[16] * 7))[0] == INVALID
    assert L.glacier_attn_cache_workspace(None, ctypes.byref(c), ctypes.byref(b), 4) == 0


def test_front_end_checks_tensors_before_the_abi():
    torch = pytest.importorskip("torch")
    kp = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    cu, lens = torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 3, dtype=torch.int32)
    good = dict(k_pages=kp, v_pages=kp.clone(), cu_tokens=cu, kv_lens=lens, page_table=table, total_tokens=1,
                max_new=0, max_kv=0, device=-1)  # -1: the device of CPU tensors
    cache, batch = ga.cache_args(**good)
    assert (cache.page_stride, cache.n_pages, cache.page_size, cache.head_dim) == (2048, 4, 16, 64)
    assert (batch.n_seqs, batch.max_pages, batch.table_stride) == (1, 3, 3)
    both = torch.zeros(4, 2, 2, 16, 64, dtype=torch.bfloat16)
    cache, _ = ga.cache_args(**dict(good, k_pages=both[:, 0], v_pages=both[:, 1]))
    assert cache.page_stride == 4096 and cache.v_pages - cache.k_pages == 4096
    wide = torch.zeros(3, 9, dtype=torch.int32)
    _, batch = ga.cache_args(**dict(good, page_table=wide[:2, :4], cu_tokens=torch.zeros(3, dtype=torch.int32),
                                    kv_lens=torch.zeros(2, dtype=torch.int32)))
    assert (batch.n_seqs, batch.max_pages, batch.table_stride) == (2, 4, 9)
    for change in (dict(k_pages=kp[0]), dict(v_pages=kp.float()), dict(v_pages=kp[:3]),
                   dict(v_pages=both[:, 1]), dict(k_pages=kp[:, :, ::2], v_pages=kp[:, :, ::2]),
                   dict(cu_tokens=lens), dict(kv_lens=cu), dict(cu_tokens=cu.long()), dict(page_table=table[0]),
                   dict(page_table=table.long()), dict(page_table=wide[:1, ::3]),
                   dict(page_table=wide[:1].expand(2, 9), cu_tokens=torch.zeros(3, dtype=torch.int32), kv_lens=cu),
                   dict(k_pages=kp.half(), v_pages=kp.half()), dict(device=0)):
        with pytest.raises(TypeError):
            ga.cache_args(**dict(good, **change))


@pytest.mark.parametrize("call", [_append, _forward])
@pytest.mark.parametrize("change,word", [
    (dict(total_tokens=1 << 26), "tensor too large"), (dict(n_seqs=1 << 21), "too many sequences"),
    (dict(n_seqs=1 << 20, n_heads_kv=8, hq=8, page_stride=8 * 16 * 64), "too many sequences"),
    (dict(hq=2 ** 31 - 2), "tensor too large"),
    (dict(n_heads_kv=2 ** 30, hq=2 ** 30, page_stride=2 ** 39, page_size=16, head_dim=8, n_pages=1),
     "tensor too large")])
def test_more_threads_than_a_launch_has(call, change, word):
    # (and head counts whose sum passes 32 bits)
    rc, msg = call(**change)
    assert rc == UNSUPPORTED and word in msg, msg


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("change", [dict(T=1 << 26, hq=1, hkv=1), dict(T=1, hq=2 ** 30), dict(T=2, hq=2 ** 29)])
def test_more_rows_than_a_norm_counts(backward, change):
    rc, msg = _norm(backward=backward, **change)
    assert rc == UNSUPPORTED and "too large" in msg, msg


PAGE = 2 * 2 * 16 * 64  # bytes of a page of _cache()


@pytest.mark.parametrize("change,word", [
    (dict(v_pages=MB), "v_pages overlaps k_pages"), (dict(v_pages=MB + PAGE), "v_pages overlaps k_pages"),
    (dict(v_pages=MB - PAGE + 16), "k_pages overlaps v_pages"), (dict(v_pages=MB + 9 * PAGE), "ctx"),
    (dict(v_pages=MB - 9 * PAGE), "ctx"), (dict(v_pages=MB + 9 * PAGE - 16), "v_pages overlaps"),
    # interleaved pages: the others' lie in the gaps
    (dict(v_pages=MB + PAGE, page_stride=PAGE), "ctx"), (dict(v_pages=MB + 3 * PAGE, page_stride=PAGE), "ctx"),
    (dict(v_pages=MB + 2 * PAGE, page_stride=PAGE), "v_pages overlaps"),
    (dict(v_pages=MB + PAGE - 16, page_stride=PAGE), "v_pages overlaps"),
    (dict(v_pages=MB + PAGE + 16, page_stride=PAGE), "v_pages overlaps"),
    (dict(k=MB + 16), "k overlaps k_pages"), (dict(v=2 * MB + 8 * PAGE), "v overlaps v_pages"),
    (dict(q=MB + PAGE), "q overlaps k_pages"), (dict(q_rot=2 * MB - 16), "q_rot overlaps v_pages"),
    (dict(k=MB + 9 * PAGE), "ctx"), (dict(k=MB - 8 * 2 * 64 * 2), "ctx"),
    (dict(k=MB + PAGE, page_stride=PAGE), "ctx"), (dict(k=MB + PAGE + 16, page_stride=2 * PAGE, v_pages=4 * MB), "ctx"),
    (dict(v_pages=MB, n_pages=0), "ctx")])
def test_append_keeps_off_the_pages(change, word):
    rc, msg = _append(**change)
    assert rc == INVALID and word in msg, msg


@pytest.mark.parametrize("change,word", [
    (dict(out=MB), "out overlaps k_pages"), (dict(lse=2 * MB + 4), "lse overlaps v_pages"),
    (dict(lse=8 * MB), "lse overlaps q"), (dict(lse=9 * MB + 64), "lse overlaps out"),
    (dict(v_pages=MB), "ctx"), (dict(q=MB), "ctx")])
def test_forward_keeps_off_the_pages(change, word):
    # (reading may share memory: one set of pages as K and V is fine)
    rc, msg = _forward(**change)
    assert rc == INVALID and word in msg, msg


@pytest.mark.parametrize("at,word", [
    ({"dk_weight": 10 * MB}, "same array"), ({"dk_weight": 10 * MB + 16}, "dq_weight overlaps dk_weight"),
    ({"dq_weight": 5 * MB}, "dq_weight overlaps q_weight"), ({"dk_weight": 6 * MB + 4}, "dk_weight overlaps k_weight"),
    ({"dk_weight": 8 * MB + 64}, "dk_weight overlaps dq"), ({"dq_weight": 10 * MB + 256}, "ctx")])
def test_weight_gradients_share_no_memory(at, word):
    rc, msg = _norm(backward=True, at=at)
    assert rc == INVALID and word in msg, msg


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("short,code,word", [(4, INVALID, "ctx"), (3, UNSUPPORTED, "too large"),
                                             (1, UNSUPPORTED, "too large")])
def test_the_longest_norm(backward, short, code, word):
    # four tokens to a workgroup of 256 threads: one more than 2^26 - 4 tokens
    # rounds up to the 2^32 threads that a launch does not have
    names = (["dq_out", "dk_out"] if backward else []) + ["q", "k", "q_weight", "k_weight", "positions"] + (
        ["dq", "dk", "dq_weight", "dk_weight"] if backward else ["q_out", "k_out"])
    rc, msg = _norm(backward=backward, T=2 ** 26 - short, hq=1, hkv=1, d=8,
                    at={n: (i + 1) << 34 for i, n in enumerate(names)})
    assert rc == code and word in msg, msg


def test_sizes_past_32_bits_are_refused_not_wrapped():
    # (descriptors hold 32-bit sizes; tensors without memory stand for the large ones)
    torch = pytest.importorskip("torch")
    import types

    bf16, i32, big = torch.bfloat16, torch.int32, 2 ** 32 + 5
    eng = types.SimpleNamespace(device_ordinal=-1, _io_of=ga.GpuAttentionEngine._io_of)
    q = torch.empty(big, 1, 8, dtype=bf16, device="meta")
    w = torch.zeros(8)
    with pytest.raises(ga.Unsupported, match="too large"):
        ga.GpuAttentionEngine._qk_args(eng, q, q, w, w, 1e-6, None, None)
    heads = torch.empty(1, big, 8, dtype=bf16, device="meta")
    with pytest.raises(ga.Unsupported, match="too large"):
        ga.GpuAttentionEngine._qk_args(eng, heads, heads, w, w, 1e-6, None, None)
    kp = torch.zeros(4, 2, 16, 64, dtype=bf16)
    good = dict(k_pages=kp, v_pages=kp.clone(), cu_tokens=torch.zeros(2, dtype=i32), kv_lens=torch.zeros(1, dtype=i32),
                page_table=torch.zeros(1, 3, dtype=i32), total_tokens=1, max_new=0, max_kv=0, device=-1)
    pages = torch.empty(big, 2, 16, 64, dtype=bf16, device="meta")
    for change in (dict(total_tokens=big), dict(total_tokens=2 ** 31),
                   dict(page_table=torch.empty(1, big, dtype=i32, device="meta")),
                   dict(k_pages=pages, v_pages=pages)):
        with pytest.raises(ga.Unsupported, match="too large"):
            ga.cache_args(**dict(good, **change))
    _, batch = ga.cache_args(**dict(good, max_new=big, max_kv=2 ** 40))  # (hints: any size is fine)
    assert batch.max_new == batch.max_kv == 2 ** 31 - 1
