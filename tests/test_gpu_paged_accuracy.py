"""Exact decode attention where errors could pile up or be hidden: long sequences far from zero, caps of any size, values that are not
finite beside others that are.  Pools whose logits are exact in 32 bits, against 64 bits.

What the kernels may be off by, from their arithmetic (u = 2^-24; T: rounds of a warp, of `keys` keys each; S parts of a unit):
* a weight exp2(s k - base), s exact: k = log2 e rounded moves it by |s - s_max| u relative (the base is common to all); the
  difference, within [-4, 16), is rounded by 2^-21, exp2 is off by 2 ulp: together below W = 2^-20;
* 16-bit products take a weight in two terms; what is left out is 2^-22 of it in half precision;
* the denominator: one rounding a round, 16 within it, S parts: (T + 16 + S) u;
* a numerator: a tensor core's step adds 16 products to the sum so far and may cut each of the 17 at the last bit of the largest:
  17 u of that sum, which grows in equal steps, so that T keys / 16 steps (twice as many where the second term is a product of its own)
  have half of 17 u each of the end; and S parts: 2 u each;
* the log-sum-exp adds the base and the logarithm of a denominator below 2^36, off by one ulp of 36: 2^-18; log2 e a itself is off by u."""
import math

import pytest
import torch

from test_gpu_paged_attention import DT, FP8

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SMS = 148


def offset_pool(n, page, HKV, D, cache_type, seed):
    """Keys (1, x_t, 0, ...) with x_t a quarter's multiple in [-1, 0]: q = (a, 1, 0, ...) gives the logit a + x_t without a rounding.  Values: even
    columns 1 in the first half of the sequence and 0 behind it, odd ones N(0, 1)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n_pages = -(-n // page)
    table = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)[None]
    t = torch.arange(n, device="cuda")
    x = torch.randint(-4, 1, (n,), generator=g, device="cuda") / 4.0
    x[n // 3] = 0.0
    v = torch.randn((n, HKV, D), generator=g, device="cuda")
    v[:, :, ::2] = (t < n // 2).float()[:, None, None]
    k = torch.zeros((n, HKV, D), device="cuda")
    k[:, :, 0], k[:, :, 1] = 1.0, x[:, None]
    caches = []
    for rows in (k, v):
        c = torch.zeros((n_pages * page, HKV, D), device="cuda")
        c[table[0, t // page].long() * page + t % page] = rows
        caches.append(c.to(cache_type).view(n_pages, page, HKV, D))
    return caches[0], caches[1], table, x.double(), v.to(cache_type).double()


@pytest.mark.parametrize("B,n", [(40, 32768), (1, 131072)])
@pytest.mark.parametrize("G", [8, 16])
@pytest.mark.parametrize("dtype,fp8,D", [("fp16", False, 64), ("fp16", False, 128), ("bf16", True, 64), ("fp16", True, 128), ("bf16", False, 128)])
def test_an_offset_of_all_logits_changes_nothing(dtype, fp8, D, G, B, n):
    """A constant added to all logits leaves the softmax as it is and the log-sum-exp moves by it, however many rounds a sequence takes."""
    from hip_attention_b200 import paged_decode_attention
    HKV = 2
    kc, vc, table, x, v = offset_pool(n, 64, HKV, D, FP8 if fp8 else DT[dtype], seed=G + D)
    H = HKV * G
    i = torch.arange(B * H, device="cuda")
    low = torch.tensor([-16.0, -64.0, -256.0], device="cuda")[i % 3]        # largest logit to base 2: fourteen below a power of two, where the shift rounds
    a = ((low + 14.0 * ((i * 0.6180339887498949) % 1.0)) * math.log(2)).view(B, H).to(DT[dtype])
    q = torch.zeros((B, H, D), dtype=DT[dtype], device="cuda")
    q[:, :, 0], q[:, :, 1] = a, 1.0
    out, lse = paged_decode_attention(q, kc, vc, table, torch.tensor([n], device="cuda"), rows=torch.zeros(B, dtype=torch.int32, device="cuda"), return_lse=True)
    p = torch.softmax(x, 0)
    want, size = (torch.einsum("t,thd->hd", p, w).repeat_interleave(G, 0) for w in (v, v.abs()))
    want_lse = (a.double() + torch.logsumexp(x, 0)) / math.log(2)
    row = D * (1 if fp8 else 2)
    keys = 32 if row <= 128 else 16
    T = math.ceil(B * HKV * math.ceil(n / (4 * keys)) / SMS) + 1            # (at least one CTA to a multiprocessor)
    S = 4 + 3 * SMS
    weight = 2.0 ** -20
    steps = T * (keys // 16) * (1 if G == 8 else 2)
    den = (T + 16 + S) * U + weight
    two_terms = 2.0 ** -16 if dtype == "bf16" and not fp8 else 2.0 ** -22
    tol = size * (weight + two_terms + den + steps * 17 * U / 2 + 2 * S * U) + torch.finfo(q.dtype).eps / 2 * want.abs()
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), f"off by {(err / tol).max().item():.3g} of the bound"
    tol = (want_lse.abs() + a.double().abs() / math.log(2)) * 2 * U + den / math.log(2) + 2.0 ** -18
    err = (lse.double() - want_lse).abs()
    assert bool((err <= tol).all()), f"lse off by {(err / tol).max().item():.3g} of the bound"


@pytest.mark.parametrize("cap", [1e-40, 1e-3, 0.5, 30.0, 64.0, 65.0, 200.0, 1e3, 1e5, 1e20, 3e38])
@pytest.mark.parametrize("dtype,fp8,G", [("fp32", False, 4), ("fp32", False, 8), ("bf16", False, 4), ("fp16", False, 12), ("bf16", True, 4), ("fp16", True, 12)])
def test_soft_caps_of_any_size(dtype, fp8, G, cap):
    """A capped logit is off by a few roundings of itself (16-bit products with caps up to 64: of the cap); a cap far above the logits changes nothing.

    z = cap tanh(s scale / cap), s exact.  scale / cap and its product with s: 6 roundings; tanhf: 2 ulp; the product with log2 e cap: 3; 13 u < 2^-20 of z, also
    where the cap is left out (y^2 / 3 < 2^-25).  Short form: 14 u < 2^-20 of the cap besides (exp2 2 ulp, the sum, the reciprocal 1 ulp, the last product)."""
    from hip_attention_b200 import paged_decode_attention
    D, page, lens = 64, 16, [1, 2, 37, 300, 1]
    g = torch.Generator(device="cuda").manual_seed(3)
    W = max(-(-n // page) for n in lens)
    n_pages = W * len(lens)
    table = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).view(len(lens), W)
    ct = FP8 if fp8 else DT[dtype]
    kc, vc = torch.zeros((n_pages, page, 1, D), device="cuda"), torch.randn((n_pages, page, 1, D), generator=g, device="cuda")
    kc[..., 0] = torch.randint(-7, 8, kc.shape[:-1], generator=g, device="cuda") / 4.0
    kc[..., 0][kc[..., 0] == 0] = 1.0
    if fp8:
        kc[..., 0] = kc[..., 0].to(FP8).float()
    kc, vc = kc.to(ct), vc.to(ct)
    q = torch.zeros((len(lens), G, D), dtype=DT[dtype], device="cuda")
    q[:, :, 0] = 2.0 ** (torch.arange(G, device="cuda") % 4 * 3 - 5)          # logits from 2^-8 to 14
    out, lse = paged_decode_attention(q, kc, vc, table, torch.tensor(lens, device="cuda"), sm_scale=0.5, logit_softcap=cap, return_lse=True)
    cap = torch.tensor(cap, dtype=torch.float32).double().item()
    short = dtype != "fp32" and cap <= 64
    for b, n in enumerate(lens):
        k, v = (c[table[b].long()].view(torch.uint8 if fp8 else ct).reshape(-1, D)[:n].view(ct).double() for c in (kc, vc))
        for h in range(G):
            z = cap * torch.tanh(k[:, 0] * q[b, h, 0].double() * 0.5 / cap)
            ds = z.abs().max().item() * 2.0 ** -20 + (2.0 ** -20 * cap if short else 0.0)
            p = torch.softmax(z, 0)
            want, size, want_lse = p @ v, p @ v.abs(), (torch.logsumexp(z, 0) / math.log(2)).item()
            weight = 2.0 ** -20 + 2 * z.abs().max().item() * U
            two_terms = {"fp32": 0.0, "fp16": 2.0 ** -22, "bf16": 2.0 ** -22 if fp8 else 2.0 ** -16}[dtype]
            tol = size * (2 * (ds + weight) + two_terms + 100 * U) + torch.finfo(q.dtype).eps / 2 * want.abs()
            err = (out[b, h].double() - want).abs()
            assert bool((err <= tol).all()), f"{n} {h}: off by {(err / tol).max().item():.3g} of the bound"
            top = 9.0 if dtype == "fp32" else 23.0        # log2 of the denominator: off by one ulp
            tol = (ds + weight + 50 * U) / math.log(2) + 2 * U * (abs(want_lse) + top)
            assert abs(lse[b, h].item() - want_lse) <= tol, f"{n} {h}: lse off by {abs(lse[b, h].item() - want_lse) / tol:.3g} of the bound"


@pytest.mark.parametrize("width", [64, 4096])
@pytest.mark.parametrize("dtype,fp8,D", [("bf16", False, 64), ("bf16", False, 128), ("bf16", False, 256), ("fp16", False, 128), ("fp16", True, 128), ("bf16", True, 64)])
@pytest.mark.parametrize("G", [8, 9, 16, 24])
def test_what_is_not_finite_costs_its_neighbours_nothing(dtype, fp8, D, G, width):
    """One infinite and one NaN value, and a NaN in one head's query: other columns and heads keep both terms of their weights.

    Two kinds of keys with logits 0 and -1.25 in such numbers that values of +1 and -1 nearly cancel: the output is small, its rounding too, and
    a weight's rounding to one term (2^-9 of exp(-1.25) in bf16, 2^-11 in half precision, the same for all its keys) would show."""
    from hip_attention_b200 import paged_decode_attention
    n, page, HKV, w = 4000, 64, 1, math.exp(-1.25)
    g = torch.Generator(device="cuda").manual_seed(5)
    n_pages = -(-n // page)
    t = torch.arange(n, device="cuda")
    first = (t * 0.6180339887498949) % 1.0 < w / (1 + w)
    k, v = torch.zeros((n, HKV, D), device="cuda"), torch.empty((n, HKV, D), device="cuda")
    k[:, 0, 0] = torch.where(first, 0.0, -1.25)
    v[:] = torch.where(first, 1.0, -1.0)[:, None, None]
    v[:, 0, 1::2] *= -1
    clean = v.double()
    v[2501, 0, 3], v[77, 0, 5] = float("inf"), float("nan")
    table = torch.full((1, width), n_pages + 3, dtype=torch.int32, device="cuda")
    table[0, :n_pages] = torch.randperm(n_pages, generator=g, device="cuda")
    ct = FP8 if fp8 else DT[dtype]
    caches = []
    for rows in (k, v):
        c = torch.zeros((n_pages * page, HKV, D), device="cuda")
        c[table[0, t // page].long() * page + t % page] = rows
        caches.append(c.to(ct).view(n_pages, page, HKV, D))
    q = torch.zeros((1, G, D), dtype=DT[dtype], device="cuda")
    q[..., 0] = 1.0
    q[0, G - 2, 2] = float("nan")
    out, lse = paged_decode_attention(q, *caches, table, torch.tensor([n], device="cuda"), return_lse=True)
    p = torch.softmax(k[:, 0, 0].double(), 0)
    want, size = p @ clean[:, 0], p @ clean[:, 0].abs()
    heads, cols = [h for h in range(G) if h != G - 2], [d for d in range(D) if d not in (3, 5)]
    assert bool(torch.isnan(out[0, G - 2]).all()) and bool(torch.isnan(lse[0, G - 2]))
    assert bool((out[0, heads, 3] == float("inf")).all()) and bool(torch.isnan(out[0, heads, 5]).all())
    two_terms = 2.0 ** -16 if dtype == "bf16" and not fp8 else 2.0 ** -22
    steps = 2 * 2 * 63                                          # (a sequence in one CTA: 63 rounds of up to 32 keys a warp, both terms)
    tol = size * (2 * 2.0 ** -20 + two_terms + (200 + steps * 17 / 2) * U) + torch.finfo(q.dtype).eps / 2 * want.abs() + 2.0 ** -25
    err = (out[0].double() - want).abs()[heads][:, cols]
    assert bool((err <= tol[cols]).all()), f"off by {(err / tol[cols]).max().item():.3g} of the bound"
    want_lse = torch.logsumexp(k[:, 0, 0].double(), 0).item() / math.log(2)
    assert bool(((lse[0, heads].double() - want_lse).abs() <= 2.0 ** -18).all())


@pytest.mark.parametrize("width", [64, 4096])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("dtype,fp8,size", [("fp16", False, 13), ("fp16", False, 15), ("fp16", True, 13), ("bf16", True, 13), ("bf16", False, 16), ("bf16", False, 60), ("fp32", False, 60)])
@pytest.mark.parametrize("G", [4, 12])
def test_logits_whose_neighbours_are_far_apart(dtype, fp8, size, sign, G, width):
    """Logits of 2^26 and beyond: the largest take all of the weight, in equal parts.  (1.25 2^size times 2^size, next to it 1 2^size times that: no
    other key is less than 2^24 below.)"""
    from hip_attention_b200 import paged_decode_attention
    n, page, D = 3000, 64, 64
    g = torch.Generator(device="cuda").manual_seed(size)
    n_pages = -(-n // page)
    t = torch.arange(n, device="cuda")
    top = torch.rand(n, generator=g, device="cuda") < 0.02
    k = torch.zeros((n, 1, D), device="cuda")
    k[:, 0, 0] = torch.where(top, 1.25 if sign > 0 else 1.0, 1.0 if sign > 0 else 1.25) * 2.0 ** size * sign
    v = torch.randn((n, 1, D), generator=g, device="cuda")
    table = torch.full((1, width), 0, dtype=torch.int32, device="cuda")
    table[0, :n_pages] = torch.randperm(n_pages, generator=g, device="cuda")
    ct = FP8 if fp8 else DT[dtype]
    caches = []
    for rows in (k, v):
        c = torch.zeros((n_pages * page, 1, D), device="cuda")
        c[table[0, t // page].long() * page + t % page] = rows
        caches.append(c.to(ct).view(n_pages, page, 1, D))
    q = torch.zeros((1, G, D), dtype=DT[dtype], device="cuda")
    q[..., 0] = 2.0 ** size * (1 + torch.arange(G, device="cuda") / 16)
    out, lse = paged_decode_attention(q, *caches, table, torch.tensor([n], device="cuda"), return_lse=True)
    vt = v.to(ct).double()[top, 0]
    want, size_ = vt.mean(0), vt.abs().mean(0)
    # weights of the largest are equal; numerators and denominators: 24 rounds, up to 300 parts (2 u each), two terms of 16 bits or one of eight bits more
    tol = size_ * ((24 * 2 * 17 + 600) * U + (2.0 ** -16 if dtype == "bf16" and not fp8 else 0.0) + 2.0 ** -20) + torch.finfo(q.dtype).eps / 2 * want.abs()
    err = (out[0].double() - want).abs()
    assert bool((err <= tol).all()), f"off by {(err / tol).max().item():.3g} of the bound"
    want_lse = q[0, :, 0].double() * k.to(ct).double()[top, 0, 0][0] / math.log(2) + math.log2(vt.shape[0])
    assert bool(((lse[0].double() - want_lse).abs() <= want_lse.abs() * 2.0 ** -21).all())


@pytest.mark.parametrize("cap", [None, 30.0, 1000.0])
@pytest.mark.parametrize("scale,query", [(1e-9, 2.0 ** -126), (1e-30, 2.0 ** -100), (1.4e-45, 1.0), (-1e-9, 2.0 ** -126), (3.4e38, 0.0), (0.0, 1.0)])
@pytest.mark.parametrize("dtype,fp8", [("bf16", True), ("fp16", True), ("bf16", False), ("fp32", False)])
def test_scales_at_the_ends_of_their_range(dtype, fp8, scale, query, cap):
    """Logits that are zero, or nothing beside 1, give the mean of the values."""
    from hip_attention_b200 import paged_decode_attention
    n, D = 500, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    ct = FP8 if fp8 else DT[dtype]
    k, v = (torch.randn((n, 1, 1, D), generator=g, device="cuda").to(ct) for _ in range(2))
    q = torch.full((1, 8, D), query, device="cuda").to(DT[dtype])
    q[0, 1] *= -1
    out, lse = paged_decode_attention(q, k, v, torch.arange(n, device="cuda")[None], torch.tensor([n], device="cuda"), sm_scale=scale, logit_softcap=cap, return_lse=True)
    want, size = v.double().mean(0)[0], v.double().abs().mean(0)[0]
    # weights are equal; the log-sum-exp: with the shift of half-precision weights, 14 + log2 500 < 23, one ulp; caps up to 64 in 16 bits: 2^-20 of the cap
    short = 2.0 ** -20 * cap if cap and cap <= 64 and dtype != "fp32" else 0.0
    tol = size * (100 * U + (2.0 ** -16 if dtype == "bf16" and not fp8 else 2.0 ** -22) + 2.0 ** -20 + 2 * short) + torch.finfo(q.dtype).eps / 2 * want.abs()
    assert bool(((out[0].double() - want).abs() <= tol).all())
    assert bool(((lse.double() - math.log2(n)).abs() <= 2.0 ** -18 + 1.5 * short).all())


@pytest.mark.parametrize("lens,width", [([300, 0, 2000, 64, 1, 777, 5000, 33] * 5, 4096), ([700, 0, 90, 1300], 96), ([40] * 200, 4)])
@pytest.mark.parametrize("dtype,fp8,D,H,HKV", [("bf16", False, 128, 32, 2), ("fp16", False, 64, 24, 2), ("bf16", True, 128, 16, 1), ("bf16", False, 256, 16, 1), ("fp16", True, 96, 48, 2),
                                               ("bf16", False, 128, 16, 2), ("fp32", False, 64, 16, 2)])
def test_other_columns_heads_and_sequences_keep_their_bits(dtype, fp8, D, H, HKV, lens, width):
    """Values that are not finite in some columns of one KV head, NaN keys in one sequence: all else comes out bit for bit as without them."""
    from hip_attention_b200 import paged_decode_attention
    page = 16
    g = torch.Generator(device="cuda").manual_seed(2)
    need = [-(-n // page) for n in lens]
    n_pages = sum(need)
    table = torch.zeros((len(lens), width * 16 // page), dtype=torch.int32, device="cuda")
    order, at = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32), 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    kc, vc = (torch.randn((n_pages, page, HKV, D), generator=g, device="cuda") for _ in range(2))
    ct = FP8 if fp8 else DT[dtype]
    sl = torch.tensor(lens, device="cuda")
    q = torch.randn((len(lens), H, D), generator=g, device="cuda").to(DT[dtype])
    call = lambda: paged_decode_attention(q, kc.to(ct), vc.to(ct), table, sl, sm_scale=D ** -0.5, return_lse=True)   # noqa: E731
    want, want_lse = call()
    vc[torch.rand(n_pages, generator=g, device="cuda") < 0.3, 5, HKV - 1, 3] = float("inf")
    vc[torch.rand(n_pages, generator=g, device="cuda") < 0.3, 9, HKV - 1, D - 1] = float("nan")
    bad = next(b for b, n in enumerate(lens) if n >= 40)
    kc[table[bad, 1].long(), 4, 0, 1] = float("nan")
    got, lse = call()
    G = H // HKV
    ok = torch.ones(got.shape, dtype=torch.bool, device="cuda")
    ok[:, (HKV - 1) * G:, 3] = ok[:, (HKV - 1) * G:, D - 1] = False
    ok[bad, :G] = False
    assert torch.equal(got[ok], want[ok]) and bool(torch.isnan(got[bad, :G]).all()) and bool(torch.isnan(lse[bad, :G]).all())
    keep = torch.ones(lse.shape, dtype=torch.bool, device="cuda")
    keep[bad, :G] = False
    assert torch.equal(lse[keep], want_lse[keep])
    assert not bool(torch.isnan(got[:, (HKV - 1) * G:, 3][keep[:, (HKV - 1) * G:]]).any())       # infinite or finite, no NaN
