"""Each refusal of the page pool's operators says what it refuses: the message names the cause, not only the code.  No GPU is needed."""
import ctypes as C

import pytest

from test_paged_refusals import _decode, _tokens


def _message():
    from hip_attention_b200 import _lib as L
    return L.load().hipattn_error_string().decode()


@pytest.mark.parametrize("kw, tok, words", [
    (dict(B=0), {}, "bad shape B=0"), (dict(H=5), {}, "bad shape B=2 H=5"), (dict(D=0), {}, "D=0"), (dict(dtype=7), {}, "unknown dtype 7"), (dict(D=264), {}, "264 is larger than 256"),
    (dict(n_rows=1), {}, "2 entries, but a table of 1 rows"), (dict(window=-1), {}, "window -1"), (dict(logit_softcap=-1.0), {}, "soft-cap -1"),
    (dict(logit_softcap=float("nan")), {}, "soft-cap"), (dict(sm_scale=float("nan")), {}, "scale"), (dict(sm_scale=float("-inf")), {}, "scale -inf"), (dict(logit_softcap=float("inf")), {}, "soft-cap inf"),
    (dict(q=None), {}, "q, out and status"), (dict(out=None), {}, "q, out and status"), (dict(status=None), {}, "q, out and status"), ({}, dict(cache=None), "must be page pools"),
    (dict(D=72), dict(fp8_e5m2=1), "multiple of 16 bytes"), ({}, dict(fp8_e5m2=1, stride_ch=136), "16-byte boundaries"), (dict(dtype=0), dict(fp8_e5m2=1), "16-bit queries"),
    (dict(scratch=None), dict(table_width=4096), "bytes of scratch are needed"), (dict(scratch=4100, scratch_bytes=1 << 30), dict(table_width=4096), "16-byte aligned"),
])
def test_decode(kw, tok, words):
    from hip_attention_b200 import _lib as L
    p = _decode(tok, **kw)
    assert L.load().hipattn_paged_decode(C.byref(p), None) != 0 and words in _message(), _message()


@pytest.mark.parametrize("tok, words", [(dict(block_table=None), "block_table"), (dict(page_size=0), "page"), (dict(table_width=0), "table"), (dict(stride_off=129), "16"), (dict(cache=4100), "16")])
def test_decode_tokens(tok, words):
    from hip_attention_b200 import _lib as L
    p = _decode(tok)
    assert L.load().hipattn_paged_decode(C.byref(p), None) == 1
    assert _message().startswith("k") and words in _message(), _message()


@pytest.mark.parametrize("kw, tok, words", [
    (dict(N=0), {}, "bad shape N=0"), (dict(B=0), {}, "B=0"), (dict(N=3), {}, "3 tokens are not a multiple of 2"), (dict(n_rows=1), {}, "a table of 1 rows"), (dict(k=None), {}, "k, v and status"),
    (dict(status=None), {}, "k, v and status"), (dict(dtype=5), {}, "unknown dtype 5"), (dict(k=4100), {}, "rows of k and v"), (dict(k_stride_t=129), {}, "rows of k and v"),
    ({}, dict(cache=None), "page pools"),
])
def test_write(kw, tok, words):
    from hip_attention_b200 import _lib as L
    p = L.WriteKvParams()
    p.k = p.v = p.status = 4096
    p.k_stride_t = p.v_stride_t = 256
    p.k_stride_h = p.v_stride_h = 128
    p.k_pool, p.v_pool = _tokens(**tok), _tokens(**tok)
    p.N, p.dtype, p.D, p.B, p.HKV, p.n_rows = 2, L.BF16, 128, 2, 2, 2
    for k, v in kw.items():
        setattr(p, k, v)
    assert L.load().hipattn_write_kv(C.byref(p), None) != 0 and "write_kv" in _message() and words in _message(), _message()


@pytest.mark.parametrize("kw, words", [
    (dict(ref_counts=None), "ref_counts"), (dict(status=None), "status"), (dict(n_pages=0), "n_pages 0"), (dict(page_size=0), "page_size 0"), (dict(n_sequences=0), "n_sequences 0"),
    (dict(table_width=0), "table_width 0"), (dict(n_sequences=262145), "262145 sequences"), (dict(n_caches=0), "0 caches"), (dict(n_caches=513), "513 caches"),
    (dict(page_bytes=24), "pages of 24 bytes"), (dict(page_stride=16), "16 apart"), (dict(scratch=None), "scratch is null"),
])
def test_pool(kw, words):
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
    for name, rc in (("pool_fork", lib.hipattn_pool_fork(C.byref(p), 4096, 4096, 1, None)), ("pool_compact", lib.hipattn_pool_compact(C.byref(p), None, None))):
        assert rc != 0
    assert _message().startswith("pool_compact") and words in _message(), _message()
    p.scratch = p.status = 4096
    for n in (0, 4097):
        if not kw.keys() - {"page_bytes", "page_stride", "n_caches", "scratch"}:
            assert lib.hipattn_pool_extend(C.byref(p), 4096, 4096, 0, n, None) == 1 and f"pool_extend: {n} entries" in _message()
            assert lib.hipattn_pool_free(C.byref(p), 4096, n, None) == 1 and f"pool_free: {n} entries" in _message()
