"""Exact decode attention over a page pool against a 64-bit computation written from the formula.

Error bound, element by element, before the first run.  With u = 2^-24, s a logit in 64 bits, A = sum_t p_t |v_t| / sum_t p_t:
* a logit is a sum of D exact or once-rounded products in 32 bits, scaled and multiplied by log2 e (and through tanh, whose
  slope is at most 1): ds <= (2 D u + 2^-21) max_t scale sum_d |q_d k_d| covers them, the accumulation of a tensor core (which
  may cut instead of round: 2 u a step) included, plus 2^-20 cap for the tanh;
* a weight exp2(x - max) has the relative error ds + |x| 2^-23 (the rounding of the product with log2 e, |x| <= S) + 2^-21 (exp2);
  16-bit types: the weights go to the tensor cores in two 16-bit terms, what is left out is at most 2^-16;
* n weights and products are added in 32 bits: n u;
numerator and denominator have that error each: |o - o'| <= 2 (ds + S 2^-22 + 2^-20 + [2^-16] + n u) A, and the output's rounding
adds eps / 2 |o|.  The log-sum-exp: log2 e (ds + S 2^-22 + 2^-20 + n u) + 2^-22 |lse|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8 = torch.float8_e5m2


def make_pool(lens, page, HKV, D, dtype, fp8=False, seed=0, spare=3, width=None, index=torch.int32, layout="plain", fill=float("nan")):
    """A pool whose every row that no sequence has is `fill`; pages in random order; table entries behind a sequence are out of range."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g, device="cuda")
    width = width or max(1, max(need))
    table = torch.full((len(lens), width), n_pages + 7, dtype=index, device="cuda")
    shape = (n_pages, page, HKV, D)
    ct = FP8 if fp8 else DT[dtype]
    if layout == "plain":
        kc, vc = torch.empty(shape, dtype=ct, device="cuda"), torch.empty(shape, dtype=ct, device="cuda")
    elif layout == "interleaved":       # K and V of a page next to one another
        both = torch.empty((n_pages, 2, page, HKV, D), dtype=ct, device="cuda")
        kc, vc = both[:, 0], both[:, 1]
    else:                               # heads outside the tokens of a page, V with a gap between its pages
        kc = torch.empty((n_pages, HKV, page, D), dtype=ct, device="cuda").transpose(1, 2)
        vc = torch.empty((n_pages, 2, HKV, page, D), dtype=ct, device="cuda")[:, 1].transpose(1, 2)
    full = torch.full(shape, fill, device="cuda").to(ct)
    for c in (kc, vc):
        (c.view(torch.uint8) if fp8 else c).copy_(full.view(torch.uint8) if fp8 else full)
    at, keys, vals = 0, [], []
    for b, n in enumerate(lens):
        pages = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = pages.to(index)
        t = torch.arange(n, device="cuda")
        pair = []
        for c in (kc, vc):
            x = torch.randn((n, HKV, D), generator=g, device="cuda").to(ct)
            if n:
                (c.view(torch.uint8) if fp8 else c)[pages[t // page], t % page] = x.view(torch.uint8) if fp8 else x
            pair.append(x.double())
        keys.append(pair[0])
        vals.append(pair[1])
    return kc, vc, table, torch.tensor(lens, dtype=index, device="cuda"), keys, vals


def reference(q, keys, vals, scale, window=None, cap=None, sixteen=True):
    """(out, lse, bound of out without its rounding, bound of lse), 64 bits."""
    B, H, D = q.shape
    out, A = torch.zeros((B, H, D), dtype=torch.float64, device=q.device), torch.zeros((B, H, D), dtype=torch.float64, device=q.device)
    lse, rel = torch.full((B, H), -math.inf, dtype=torch.float64, device=q.device), torch.zeros((B, H), dtype=torch.float64, device=q.device)
    for b in range(B):
        n = keys[b].shape[0]
        if n == 0:
            continue
        lo = max(0, n - window) if window else 0
        k, v = keys[b][lo:], vals[b][lo:]
        G = H // k.shape[1]
        for h in range(H):
            kk, vv = k[:, h // G], v[:, h // G]
            x = kk @ q[b, h].double() * scale
            mag = (kk.abs() @ q[b, h].double().abs()).max().item() * abs(scale)
            ds = (2 * D * 2.0 ** -24 + 2.0 ** -21) * mag
            if cap:
                x = torch.tanh(x / cap) * cap
                ds += 2.0 ** -20 * cap
            p = torch.softmax(x, 0)
            out[b, h], A[b, h] = p @ vv, p @ vv.abs()
            lse[b, h] = torch.logsumexp(x, 0) / math.log(2)
            rel[b, h] = ds + x.abs().max().item() * 2.0 ** -22 + 2.0 ** -20 + kk.shape[0] * 2.0 ** -24
    return out, lse, 2 * (rel + (2.0 ** -16 if sixteen else 0.0))[..., None] * A, rel / math.log(2) + lse.abs().nan_to_num(0, 0, 0) * 2.0 ** -22


def check(got, lse, ref, dtype):
    out, want, bound, bound_lse = ref
    err = (got.double() - out).abs()
    tol = bound + torch.finfo(dtype).eps / 2 * out.abs() + torch.finfo(dtype).tiny
    assert bool((err <= tol).all()), f"off by {(err / tol).max().item():.3g} of the bound"
    if lse is not None:
        assert torch.equal(torch.isinf(lse), torch.isinf(want))
        fine = torch.isfinite(want)
        err = (lse.double() - want).abs()[fine]
        assert bool((err <= bound_lse[fine]).all()), f"lse off by {(err / bound_lse[fine]).max().item():.3g} of the bound"


def run(lens, page, H, HKV, D, dtype, fp8=False, window=None, cap=None, rows=False, index=torch.int32, layout="plain", seed=0, scale=None, width=None):
    from hip_attention_b200 import paged_decode_attention, read_status
    kc, vc, table, sl, keys, vals = make_pool(lens, page, HKV, D, dtype, fp8, seed, index=index, layout=layout, width=width)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    scale = D ** -0.5 if scale is None else scale
    who = list(range(len(lens)))
    if rows:
        who = [len(lens) - 1, -1, 0, 0, -5] + who
    q = torch.randn((len(who), H, D), generator=g, device="cuda").to(DT[dtype])
    read_status("cuda")
    r = torch.tensor(who, dtype=index, device="cuda") if rows else None
    got, lse = paged_decode_attention(q, kc, vc, table, sl, rows=r, sm_scale=scale, sliding_window=window, logit_softcap=cap, return_lse=True)
    assert read_status("cuda") == 0
    none = torch.zeros((0, HKV, D), dtype=torch.float64, device="cuda")
    ref = reference(q, [keys[i] if i >= 0 else none for i in who], [vals[i] if i >= 0 else none for i in who], scale, window, cap, dtype != "fp32")
    assert got.shape == q.shape and got.dtype == q.dtype and lse.dtype == torch.float32
    check(got, lse, ref, q.dtype)
    return q, kc, vc, table, sl, got, lse


EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1025]


@pytest.mark.parametrize("dtype,fp8", [("bf16", False), ("fp16", False), ("fp32", False), ("bf16", True), ("fp16", True)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_lengths_at_the_edges_of_tiles(dtype, fp8, D):
    run(EDGES, 16, 8, 2, D, dtype, fp8)


@pytest.mark.parametrize("page", [1, 3, 16, 20, 64, 1000])
@pytest.mark.parametrize("dtype,fp8", [("bf16", False), ("fp32", False), ("fp16", True)])
def test_page_sizes(page, dtype, fp8):
    run([1, 777, 64, 0, 1300], page, 8, 2, 128, dtype, fp8, seed=page)


@pytest.mark.parametrize("H,HKV", [(1, 1), (4, 4), (6, 2), (5, 1), (8, 1), (28, 4), (16, 1), (17, 1), (40, 2), (64, 1), (24, 2)])
@pytest.mark.parametrize("dtype,fp8", [("bf16", False), ("fp32", False), ("bf16", True)])
def test_head_layouts(H, HKV, dtype, fp8):
    run([700, 3, 129], 16, H, HKV, 64, dtype, fp8, seed=H)


@pytest.mark.parametrize("dtype,D,fp8", [("bf16", 8, False), ("bf16", 72, False), ("fp16", 96, False), ("bf16", 136, False), ("fp32", 4, False), ("fp32", 100, False),
                                         ("fp32", 192, False), ("bf16", 248, False), ("bf16", 16, True), ("fp16", 80, True), ("bf16", 112, True), ("fp16", 240, True)])
def test_odd_head_dimensions(dtype, D, fp8):
    run([600, 1, 0, 77], 16, 4, 2, D, dtype, fp8, seed=D)


@pytest.mark.parametrize("window", [1, 15, 16, 100, 257, 5000])
@pytest.mark.parametrize("dtype,fp8", [("bf16", False), ("fp32", False), ("bf16", True)])
def test_sliding_window(window, dtype, fp8):
    run([1, 0, 100, 999, 3001], 16, 8, 2, 128, dtype, fp8, window=window)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_soft_cap_and_scale(dtype):
    run([500, 2, 1200], 16, 8, 2, 128, dtype, cap=5.0, scale=0.5)
    run([500, 2, 1200], 16, 8, 2, 128, dtype, cap=30.0)
    run([500, 2, 1200], 16, 8, 2, 64, dtype, scale=1.0)     # logits of +-30: nearly one key
    run([500, 2, 1200], 16, 8, 2, 64, dtype, scale=0.0)     # the mean
    run([500, 2, 1200], 16, 8, 2, 64, dtype, scale=-0.2)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("layout", ["plain", "interleaved", "heads_first"])
@pytest.mark.parametrize("dtype,fp8", [("bf16", False), ("fp32", False), ("fp16", True)])
def test_rows_layouts_and_index_types(index, layout, dtype, fp8):
    run([300, 0, 1, 2049], 16, 8, 2, 128, dtype, fp8, rows=True, index=index, layout=layout)


@pytest.mark.parametrize("dtype,fp8", [("bf16", False), ("fp32", False), ("bf16", True)])
@pytest.mark.parametrize("B", [1, 7, 150, 700])
def test_batches(B, dtype, fp8):
    """Batches smaller and larger than the GPU and than a block of threads; wide tables, of which little is used."""
    lens = [(i * 37) % 211 for i in range(B)]
    lens[0] = 9001
    run(lens, 16, 4, 2, 64, dtype, fp8, seed=B, width=1024)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_long_sequences(dtype):
    run([70001, 5], 64, 8, 2, 128, dtype)


@pytest.mark.parametrize("fp8", [False, True])
def test_many_equal_small_weights(fp8):
    """One key far above 60000 others, whose weights are below 2^-17 of its own each: their sum is a fair part of the output, and a
    16-bit weight that went under would show."""
    from hip_attention_b200 import paged_decode_attention
    n, D = 60001, 64
    kc, vc, table, sl, keys, vals = make_pool([n], 64, 1, D, "fp16", fp8)
    kc.view(torch.uint8 if fp8 else torch.float16).zero_()
    flat_k = kc.view(-1, 1, D)
    at = (table[0, 100].long() * 64 + 5).item()      # position 6405
    one = torch.zeros(D, device="cuda")
    one[0] = 1.0
    flat_k.view(torch.uint8 if fp8 else torch.float16)[at, 0] = one.to(kc.dtype).view(torch.uint8) if fp8 else one.half()
    keys[0].zero_()
    keys[0][6405, 0, 0] = 1.0
    q = torch.zeros((1, 2, D), dtype=torch.float16, device="cuda")
    q[0, :, 0] = torch.tensor([11.8, 9.0])
    got, lse = paged_decode_attention(q, kc, vc, table, sl, return_lse=True)
    check(got, lse, reference(q, keys, vals, 1.0), q.dtype)


@pytest.mark.parametrize("dtype,fp8", [("bf16", False), ("fp16", False), ("fp32", False), ("bf16", True)])
def test_infinities_and_nan_stay_where_they_are_attended(dtype, fp8):
    from hip_attention_b200 import paged_decode_attention
    lens = [400, 400, 400, 400]
    kc, vc, table, sl, keys, vals = make_pool(lens, 16, 1, 64, dtype, fp8)
    slot = [int(table[b, 333 // 16]) for b in range(4)]
    bits = (lambda c: c.view(torch.uint8)) if fp8 else (lambda c: c)
    put = (lambda x: torch.tensor(x, device="cuda").to(FP8).view(torch.uint8)) if fp8 else (lambda x: x)
    bits(vc)[slot[0], 333 % 16, 0, 3] = put(float("inf"))
    bits(vc)[slot[1], 333 % 16, 0, 3] = put(float("nan"))
    bits(kc)[slot[2], 333 % 16, 0, 3] = put(float("nan"))
    q = torch.ones((4, 2, 64), dtype=DT[dtype], device="cuda")
    got, lse = paged_decode_attention(q, kc, vc, table, sl, sm_scale=0.1, return_lse=True)
    rest = [i for i in range(64) if i != 3]
    assert bool((got[0, :, 3] == float("inf")).all()) and bool(torch.isfinite(got[0][:, rest]).all())
    assert bool(torch.isnan(got[1, :, 3]).all()) and bool(torch.isfinite(got[1][:, rest]).all())
    assert bool(torch.isnan(got[2]).all()) and bool(torch.isnan(lse[2]).all())
    assert bool(torch.isfinite(got[3]).all()) and bool(torch.isfinite(lse[[0, 1, 3]]).all())
    # outside the window they do not count
    got, lse = paged_decode_attention(q, kc, vc, table, sl, sm_scale=0.1, sliding_window=60, return_lse=True)
    assert bool(torch.isfinite(got).all()) and bool(torch.isfinite(lse).all())


def test_strided_queries_and_outputs():
    from hip_attention_b200 import paged_decode_attention
    q, kc, vc, table, sl, got, _ = run([300, 17], 16, 8, 2, 128, "bf16")
    wide = torch.full((2, 24, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 8:16] = q                                          # queries inside a fused projection
    out = torch.full((2, 10, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    r = paged_decode_attention(wide[:, 8:16], kc, vc, table, sl, sm_scale=128 ** -0.5, out=out[:, 1:9])
    assert r.data_ptr() == out[:, 1:9].data_ptr() and torch.equal(r, got)
    assert bool((out[:, 0] == 3).all()) and bool((out[:, 9] == 3).all())


def test_offsets_beyond_32_bits():
    from hip_attention_b200 import paged_decode_attention
    n_pages, page = 40000, 64
    kc = torch.empty((n_pages, page, 8, 128), dtype=torch.bfloat16, device="cuda")      # 5.2 GB, 2.6 G elements
    vc = torch.empty((n_pages, page, 8, 128), dtype=torch.bfloat16, device="cuda")
    pages = torch.tensor([[39999, 5, 33000, 39998, 16383, 16384, 32768]], dtype=torch.int32, device="cuda")
    n = 7 * page - 9
    g = torch.Generator(device="cuda").manual_seed(1)
    keys, vals = [], []
    for c, to in ((kc, keys), (vc, vals)):
        x = torch.randn((7 * page, 8, 128), generator=g, device="cuda").to(torch.bfloat16)
        c[pages[0].long()] = x.view(7, page, 8, 128)
        to.append(x[:n].double())
    q = torch.randn((1, 16, 128), generator=g, device="cuda").to(torch.bfloat16)
    got, lse = paged_decode_attention(q, kc, vc, pages, torch.tensor([n], device="cuda"), sm_scale=0.1, return_lse=True)
    check(got, lse, reference(q, keys, vals, 0.1), q.dtype)


def test_status_of_what_is_out_of_range():
    """Pages outside the pool read page 0, lengths stop at the table, rows beyond it are empty; each leaves its bit."""
    from hip_attention_b200 import _lib as L, paged_decode_attention, read_status
    lens = [40, 40, 40]
    kc, vc, table, sl, keys, vals = make_pool(lens, 16, 2, 64, "bf16", fill=0.0)
    q = torch.randn((3, 4, 64), device="cuda").to(torch.bfloat16)
    read_status("cuda")
    want, _ = paged_decode_attention(q, kc, vc, table, sl, return_lse=True)
    assert read_status("cuda") == 0
    bad = table.clone()
    bad[1, 1] = kc.shape[0]
    zero = table.clone()
    zero[1, 1] = 0
    got = paged_decode_attention(q, kc, vc, bad, sl)
    assert read_status("cuda") == L.STATUS_PAGE_RANGE
    assert torch.equal(got, paged_decode_attention(q, kc, vc, zero, sl)) and torch.equal(got[[0, 2]], want[[0, 2]])
    long = sl.clone()
    long[2] = 49
    got = paged_decode_attention(q, kc, vc, table, long)
    assert read_status("cuda") == L.STATUS_TOKEN_RANGE and torch.equal(got[:2], want[:2])
    got = paged_decode_attention(q, kc, vc, table, sl, rows=torch.tensor([0, 3, 2], device="cuda"))
    assert read_status("cuda") == L.STATUS_SEQUENCE and torch.equal(got[[0, 2]], want[[0, 2]]) and not got[1].any()
    neg = sl.clone()
    neg[0] = -3
    assert not paged_decode_attention(q, kc, vc, table, neg)[0].any() and read_status("cuda") == 0


def test_refusals_of_tensors():
    from hip_attention_b200 import paged_decode_attention
    _, kc, vc, table, sl, _, _ = run([40, 40], 16, 4, 2, 64, "bf16")
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device="cuda")
    for bad in (lambda: paged_decode_attention(q[0], kc, vc, table, sl), lambda: paged_decode_attention(q.half(), kc, vc, table, sl),
                lambda: paged_decode_attention(q[:, :3], kc, vc, table, sl), lambda: paged_decode_attention(q[..., :32], kc, vc, table, sl),
                lambda: paged_decode_attention(q, kc, vc[:-1], table, sl), lambda: paged_decode_attention(q, kc, vc, table.float(), sl),
                lambda: paged_decode_attention(q, kc, vc, table, sl[:1]), lambda: paged_decode_attention(q[:1], kc, vc, table, sl),
                lambda: paged_decode_attention(q, kc, vc, table, sl.cpu()), lambda: paged_decode_attention(q, kc, vc, table, sl, rows=sl[:1]),
                lambda: paged_decode_attention(q, kc, vc, table, sl, sliding_window=0), lambda: paged_decode_attention(q, kc, vc, table, sl, logit_softcap=-1.0),
                lambda: paged_decode_attention(q, kc, vc, table, sl, out=q.float()), lambda: paged_decode_attention(q.cpu(), kc, vc, table, sl),
                lambda: paged_decode_attention(q.double(), kc, vc, table, sl), lambda: paged_decode_attention(q.transpose(1, 2), kc, vc, table, sl),
                lambda: paged_decode_attention(q, kc, vc, table, sl, sm_scale=float("nan"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        paged_decode_attention(torch.zeros((2, 4, 64), device="cuda"), kc.to(FP8), vc.to(FP8), table, sl)
    assert paged_decode_attention(q[:0], kc, vc, table, sl, rows=sl[:0]).shape == (0, 4, 64)


def test_same_call_same_bits_and_two_streams_at_once():
    """Parts are joined in order, so a call repeats bit for bit, also beside another on another stream (each has its own scratch)."""
    from hip_attention_b200 import paged_decode_attention
    args = [run([9000, 31, 1200, 5], 16, 8, 2, 128, d, seed=i)[:5] for i, d in enumerate(("bf16", "fp32"))]
    want = [paged_decode_attention(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (s, a) in enumerate(zip(streams, args)):
            with torch.cuda.stream(s):
                got[i].append(paged_decode_attention(*a))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


def test_captured_and_replayed_on_other_lengths():
    from hip_attention_b200 import paged_decode_attention
    lens = [9000, 31, 1200, 5]
    q, kc, vc, table, sl, _, _ = run(lens, 16, 8, 2, 128, "bf16")
    graphs = []
    for _ in range(2):      # two graphs alive at once
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = paged_decode_attention(q, kc, vc, table, sl, sm_scale=0.1)
        graphs.append((gr, out))
    for new in ([9000, 31, 1200, 5], [1, 31, 0, 5], [8999, 0, 3, 5]):
        sl.copy_(torch.tensor(new))
        want = paged_decode_attention(q, kc, vc, table, sl, sm_scale=0.1)
        for gr, out in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)


@pytest.mark.parametrize("D", [64, 96])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_pools_whose_tokens_lie_further_apart_than_their_pages(dtype, D):
    """[page_size, n_pages, kv_heads, head_dim] seen as pages."""
    from hip_attention_b200 import paged_decode_attention
    lens = [300, 1, 77]
    kc, vc, table, sl, keys, vals = make_pool(lens, 16, 2, D, dtype)
    turned = [c.transpose(0, 1).contiguous().transpose(0, 1) for c in (kc, vc)]
    assert turned[0].stride(1) > turned[0].stride(0)
    q = torch.randn((3, 4, D), device="cuda").to(DT[dtype])
    got, lse = paged_decode_attention(q, *turned, table, sl, sm_scale=0.1, return_lse=True)
    check(got, lse, reference(q, keys, vals, 0.1, sixteen=dtype != "fp32"), q.dtype)
    assert torch.equal(got, paged_decode_attention(q, kc, vc, table, sl, sm_scale=0.1))
