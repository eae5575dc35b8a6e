"""What the page pool's operators refuse before anything is launched: no GPU is needed."""
import ctypes as C

import pytest
import torch


def _tokens(**kw):
    from hip_attention_b200 import _lib as L
    t = L.Tokens()
    t.cache, t.block_table, t.cache_seq_lens = 4096, 4096, 4096       # (never read: every call here is refused)
    t.stride_page, t.stride_off, t.stride_ch = 4 * 2 * 128, 2 * 128, 128
    t.n_pages, t.table_width, t.page_size, t.table_stride_b = 8, 4, 4, 4
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def _decode(tok=None, **kw):
    from hip_attention_b200 import _lib as L
    p = L.PagedDecodeParams()
    p.q = p.out = p.status = p.scratch = 4096
    p.k, p.v = _tokens(**(tok or {})), _tokens(**(tok or {}))
    p.dtype, p.D, p.B, p.H, p.HKV, p.n_rows, p.sm_scale = L.BF16, 128, 2, 4, 2, 2, 1.0
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw, tok, code", [
    (dict(B=0), {}, 1), (dict(H=5), {}, 1), (dict(D=0), {}, 1), (dict(dtype=7), {}, 1), (dict(D=264), {}, 2), (dict(D=68), {}, 1),
    (dict(n_rows=1), {}, 1), (dict(window=-1), {}, 1), (dict(logit_softcap=-1.0), {}, 1), (dict(logit_softcap=float("nan")), {}, 1),
    (dict(sm_scale=float("nan")), {}, 1), (dict(sm_scale=float("-inf")), {}, 1), (dict(logit_softcap=float("inf")), {}, 1), (dict(q=None), {}, 1), (dict(out=None), {}, 1), (dict(status=None), {}, 1),
    ({}, dict(cache=None), 1), ({}, dict(block_table=None), 1), ({}, dict(page_size=0), 1), ({}, dict(table_width=0), 1),
    ({}, dict(stride_off=129), 1), ({}, dict(cache=4100), 1), (dict(dtype=0), dict(fp8_e5m2=1), 2), (dict(D=72), dict(fp8_e5m2=1), 2),
    ({}, dict(fp8_e5m2=1, stride_ch=136), 2),
    (dict(scratch=None), dict(table_width=4096), 1), (dict(scratch=4100, scratch_bytes=1 << 30), dict(table_width=4096), 1),
])
def test_decode_refusals(kw, tok, code):
    from hip_attention_b200 import _lib as L
    p = _decode(tok, **kw)
    assert L.load().hipattn_paged_decode(C.byref(p), None) == code
    assert b"paged_decode" in L.load().hipattn_error_string() or b": " in L.load().hipattn_error_string()


def test_decode_refuses_null_and_unequal_pools():
    from hip_attention_b200 import _lib as L
    lib = L.load()
    assert lib.hipattn_paged_decode(None, None) == 1
    for field, value in (("n_pages", 9), ("page_size", 8), ("fp8_e5m2", 1)):
        p = _decode()
        setattr(p.v, field, value)
        assert lib.hipattn_paged_decode(C.byref(p), None) == 1


def test_decode_scratch_reads_shapes_only():
    from hip_attention_b200 import _lib as L
    lib = L.load()
    assert lib.hipattn_paged_decode_scratch(C.byref(_decode())) == 0                       # sixteen positions: not cut
    assert lib.hipattn_paged_decode_scratch(C.byref(_decode(dict(table_width=4096)))) > 0
    assert lib.hipattn_paged_decode_scratch(C.byref(_decode(dict(table_width=4096), window=8))) == 0
    assert lib.hipattn_paged_decode_scratch(C.byref(_decode(B=0))) == 0


@pytest.mark.parametrize("kw, tok, code", [
    (dict(N=0), {}, 1), (dict(B=0), {}, 1), (dict(N=3), {}, 1), (dict(n_rows=1), {}, 1), (dict(k=None), {}, 1), (dict(status=None), {}, 1),
    (dict(dtype=5), {}, 1), (dict(k=4100), {}, 1), (dict(k_stride_t=129), {}, 1), (dict(dtype=0), dict(fp8_e5m2=1), 2), ({}, dict(cache=None), 1),
    (dict(D=100), {}, 1),
])
def test_write_refusals(kw, tok, code):
    from hip_attention_b200 import _lib as L
    p = L.WriteKvParams()
    p.k = p.v = p.status = 4096
    p.k_stride_t = p.v_stride_t = 256
    p.k_stride_h = p.v_stride_h = 128
    p.k_pool, p.v_pool = _tokens(**tok), _tokens(**tok)
    p.N, p.dtype, p.D, p.B, p.HKV, p.n_rows = 2, L.BF16, 128, 2, 2, 2
    for k, v in kw.items():
        setattr(p, k, v)
    assert L.load().hipattn_write_kv(C.byref(p), None) == code
    assert L.load().hipattn_write_kv(None, None) == 1


@pytest.mark.parametrize("kw", [
    dict(ref_counts=None), dict(seq_lens=None), dict(block_table=None), dict(status=None), dict(n_pages=0), dict(page_size=0), dict(n_sequences=0),
    dict(table_width=0), dict(n_caches=0), dict(n_caches=513), dict(page_bytes=0), dict(page_bytes=24), dict(page_stride=16), dict(page_stride=1030), dict(scratch=None),
])
def test_pool_refusals(kw):
    from hip_attention_b200 import _lib as L
    lib = L.load()
    caches = (C.c_void_p * 2)(4096, 8192)
    p = L.PagePool()
    p.ref_counts = p.seq_lens = p.block_table = p.status = p.scratch = 4096
    p.caches = C.cast(caches, C.POINTER(C.c_void_p))
    p.page_stride = p.page_bytes = 1024
    p.n_pages, p.page_size, p.n_sequences, p.table_width, p.n_caches = 8, 4, 3, 4, 2
    for k, v in kw.items():
        setattr(p, k, v)
    assert lib.hipattn_pool_fork(C.byref(p), 4096, 4096, 1, None) == 1
    assert lib.hipattn_pool_compact(C.byref(p), None, None) == 1
    if set(kw) & {"ref_counts", "seq_lens", "block_table", "status", "n_pages", "page_size", "n_sequences", "table_width"}:
        assert lib.hipattn_pool_extend(C.byref(p), 4096, 4096, 0, 1, None) == 1
        assert lib.hipattn_pool_free(C.byref(p), 4096, 1, None) == 1


def test_pool_calls_refuse_bad_entries():
    from hip_attention_b200 import _lib as L
    lib = L.load()
    p = L.PagePool()
    p.ref_counts = p.seq_lens = p.block_table = p.status = p.scratch = 4096
    p.n_pages, p.page_size, p.n_sequences, p.table_width = 8, 4, 3, 4
    for n in (0, -1, 4097):
        assert lib.hipattn_pool_extend(C.byref(p), 4096, 4096, 0, n, None) == 1
        assert lib.hipattn_pool_free(C.byref(p), 4096, n, None) == 1
    assert lib.hipattn_pool_extend(C.byref(p), None, 4096, 0, 1, None) == 1
    assert lib.hipattn_pool_free(C.byref(p), None, 1, None) == 1
    assert lib.hipattn_pool_extend(None, 4096, 4096, 0, 1, None) == 1 and lib.hipattn_pool_free(None, 4096, 1, None) == 1


def test_host_tensors_are_refused():
    from hip_attention_b200 import HiPPagePool, paged_decode_attention, write_paged_kv
    cache = torch.zeros((4, 4, 2, 64))
    table, lens = torch.zeros((1, 2), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        paged_decode_attention(torch.zeros((1, 4, 64)), cache, cache.clone(), table, lens)
    with pytest.raises(ValueError):
        write_paged_kv(torch.zeros((1, 2, 64)), torch.zeros((1, 2, 64)), cache, cache.clone(), table, lens)
    with pytest.raises(ValueError):
        HiPPagePool([cache], [cache.clone()], 2, 2)
    with pytest.raises(ValueError):
        HiPPagePool([], [], 2, 2)


def test_structures_match_the_header():
    """ctypes structures list the header's fields in the header's order."""
    import os
    import re
    from hip_attention_b200 import _lib as L
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "include", "hipattn.h")) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    for name, cls in (("hipattn_paged_decode_params", L.PagedDecodeParams), ("hipattn_write_kv_params", L.WriteKvParams), ("hipattn_page_pool", L.PagePool)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s_t;" % (name, name), text, flags=re.S).group(1)
        fields = []
        for decl in body.split(";"):
            names = re.sub(r"^\s*(const\s+)?\w+", "", decl.strip()).replace("const", "")
            fields += [n.strip().lstrip("* ").strip() for n in names.split(",") if n.strip()]
        assert fields == [f[0] for f in cls._fields_], name
