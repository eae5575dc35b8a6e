"""The operators of a page pool: what a server calls next to the sparse attention of a layer, over the range of sizes it calls them at.

* ``attend``  exact attention of one new token a sequence over its pages (layers that are kept dense);
* ``write``   the keys and values of new tokens into their pages, one layer;
* ``beam``    a step of beam search: the losing beams are freed and forked anew from the winners (shared pages are counted,
  the begun page of a beam is copied in all layers);
* ``admit``   finished sequences are freed and the requests that take their places are given pages;
* ``compact`` pages in use move to the front of the pool, in all layers and tables.

Plain forms are elementary torch operations in 32 bits.  Pools hold N(0, 1) values; pages are dealt out in random order, as they
are in a pool that has been in use.  Caches that are only copied are returned as the bits they hold.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FP8 = torch.float8_e5m2


def listed():
    return [
        # The smallest call: one chat, a few hundred tokens.  Made once per layer and token: latency.
        dict(name="attend_one_short", kind="attend", B=1, T=389, ragged=False, page=16, H=16, HKV=4, D=64, dtype="fp16", fp8=False, window=0, softcap=0.0),
        # A batch of chats of very different lengths, one place of the batch empty.
        dict(name="attend_ragged_batch", kind="attend", B=32, T=16384, ragged=True, page=64, H=32, HKV=8, D=128, dtype="bf16", fp8=False, window=0, softcap=0.0),
        # A server's token-granular fp8 pool, soft-capped logits.
        dict(name="attend_server_fp8", kind="attend", B=12, T=40961, ragged=True, page=1, H=32, HKV=8, D=128, dtype="bf16", fp8=True, window=0, softcap=30.0),
        # One sequence of a million tokens.
        dict(name="attend_one_1m", kind="attend", B=1, T=1048571, ragged=False, page=64, H=32, HKV=8, D=128, dtype="bf16", fp8=False, window=0, softcap=0.0),
        # The new tokens of a decode step.
        dict(name="write_step", kind="write", B=32, n=1, T=4096, ragged=False, page=64, HKV=8, D=128, dtype="bf16", fp8=False),
        # Prompts of different lengths into an fp8 pool of single tokens.
        dict(name="write_prompts_fp8", kind="write", B=7, n=4001, T=8192, ragged=True, page=1, HKV=8, D=128, dtype="bf16", fp8=True),
        # One request of four beams, a small model.
        dict(name="beam_one", kind="beam", requests=1, beams=4, T=701, page=16, layers=2, HKV=4, D=64, dtype="fp16"),
        # A batch of requests, all layers of a larger model.
        dict(name="beam_batch", kind="beam", requests=32, beams=4, T=509, page=64, layers=16, HKV=8, D=128, dtype="bf16"),
        # A few requests into a pool of pages of sixteen.
        dict(name="admit_few", kind="admit", R=16, n=3, T=1021, page=16, pages=2048),
        # A token-granular pool: every token is a page.
        dict(name="admit_tokens", kind="admit", R=96, n=24, T=2999, page=1, pages=262144),
        # A small pool after a few sequences have ended.
        dict(name="compact_small", kind="compact", R=16, T=301, page=16, layers=2, HKV=4, D=64, dtype="fp16"),
        # A large one, all layers: before a pool is shrunk.
        dict(name="compact_large", kind="compact", R=48, T=2003, page=64, layers=8, HKV=8, D=128, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend"] * 5 + ["write", "beam", "admit", "compact"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "attend":
        H, HKV = rng.choice([(32, 8), (32, 8), (64, 8), (16, 4), (28, 4), (8, 8), (16, 1)])
        D = rng.choice([128, 128, 64, 96, 256])
        B = _log_int(rng, 1, 64)
        row = 2 * HKV * D * 4                                   # (K and V of a token in 32 bits, as the plain form holds them)
        most = max(2, min(524288, (4 << 30) // (row * B)))
        T = _log_int(rng, min(rng.choice([1, 200, 2000]), most // 2), most)
        return dict(kind=kind, B=B, T=T, ragged=rng.random() < 0.5, page=rng.choice([1, 16, 64, 20]), H=H, HKV=HKV, D=D, dtype=dtype,
                    fp8=dtype != "fp32" and rng.random() < 0.3, window=rng.choice([0, 0, 0, 1024, 257]), softcap=rng.choice([0.0, 0.0, 0.0, 30.0]))
    HKV, D = rng.choice([(8, 128), (8, 128), (4, 64), (2, 96)])
    page = rng.choice([1, 16, 64, 20])
    if kind == "write":
        n, B = _log_int(rng, 1, 4096), _log_int(rng, 1, 48)
        n = max(1, min(n, 65536 // B))
        return dict(kind=kind, B=B, n=n, T=n + _log_int(rng, 1, 2048), ragged=rng.random() < 0.5, page=page, HKV=HKV, D=D, dtype=dtype,
                    fp8=dtype != "fp32" and rng.random() < 0.4)
    if kind == "beam":
        return dict(kind=kind, requests=_log_int(rng, 1, 24), beams=rng.choice([2, 4, 5]), T=_log_int(rng, 2, 509), page=rng.choice([16, 64, 20]),
                    layers=_log_int(rng, 1, 16), HKV=HKV, D=D, dtype=dtype if dtype != "fp32" else "bf16")
    if kind == "admit":
        R = _log_int(rng, 4, 128)
        T = _log_int(rng, 2, 4096)
        return dict(kind=kind, R=R, n=max(1, R // rng.choice([1, 2, 4])), T=T, page=page, pages=R * (-(-T // page)) + _log_int(rng, 8, 65536))
    return dict(kind=kind, R=_log_int(rng, 2, 48), T=_log_int(rng, 2, 2003), page=rng.choice([16, 64, 20]), layers=_log_int(rng, 1, 6), HKV=HKV, D=D,
                dtype=dtype if dtype != "fp32" else "bf16")


# ---------------------------------------------------------------------------------------------------------------------
# sizes that follow from a case alone
# ---------------------------------------------------------------------------------------------------------------------
def _spread(n, T, empty=False):
    """n lengths up to T, spread over [T / 8, T], the first of them T; with `empty` the last is 0."""
    lens = [max(1, T - int((i * 0.6180339887498949 % 1.0) * T * 7 / 8)) for i in range(n)]
    if empty and n > 1:
        lens[-1] = 0
    return lens


def _lengths(c):
    return _spread(c["B"], c["T"], empty=True) if c["ragged"] else [c["T"]] * c["B"]


def _new_tokens(c):
    """write: new tokens of each sequence (its length in the pool includes them)."""
    return _spread(c["B"], c["n"]) if c["ragged"] else [c["n"]] * c["B"]


def _pages(length, page):
    return -(-length // page)


def _attended(c):
    return sum(min(n, c["window"]) if c["window"] else n for n in _lengths(c))


def _kept(c):
    """compact: (lengths of all sequences, those that are still there): every third has ended."""
    lens = _spread(c["R"], c["T"])
    return lens, [n if i % 3 else 0 for i, n in enumerate(lens)]


def work(c):
    eb = 4 if c.get("dtype") == "fp32" else 2
    cb = 1 if c.get("fp8") else eb
    if c["kind"] == "attend":
        keys = _attended(c)
        return {"bytes": 2 * keys * c["HKV"] * c["D"] * cb + 2 * c["B"] * c["H"] * c["D"] * eb + 4 * c["B"] * c["H"] + 4 * _pages(keys, c["page"]),
                "flops": 4 * keys * c["H"] * c["D"]}
    if c["kind"] == "write":
        n = sum(_new_tokens(c))
        return {"bytes": 2 * n * c["HKV"] * c["D"] * (eb + cb) + 4 * n, "flops": 0}
    if c["kind"] == "beam":
        children = c["requests"] * (c["beams"] - 1)
        token = 2 * c["layers"] * c["HKV"] * c["D"] * eb
        full = c["T"] // c["page"]
        # freed: table, counts; forked: table read and written, counts; the begun page read and written
        return {"bytes": children * (c["T"] % c["page"] * token * 2 + 4 * full * 7 + 64), "flops": 0}
    if c["kind"] == "admit":
        lens = _spread(c["R"], c["T"])[:c["n"]]
        return {"bytes": 4 * c["pages"] + 5 * 4 * sum(_pages(n, c["page"]) for n in lens), "flops": 0}
    lens, kept = _kept(c)
    total, live = sum(_pages(n, c["page"]) for n in lens), sum(_pages(n, c["page"]) for n in kept)
    moved = live * (total - live) / total            # (pages lie in random order)
    return {"bytes": 2 * moved * c["page"] * 2 * c["layers"] * c["HKV"] * c["D"] * eb + 4 * total + 8 * live, "flops": 0}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _tables(lens, page, n_pages, g, rows=None, width=None):
    """A block table and lengths on the GPU, the pages in random order; `rows`: places of the sequences in the table."""
    dev = "cuda"
    need = torch.tensor([_pages(n, page) for n in lens], device=dev)
    order = torch.randperm(n_pages, generator=g, device=dev)
    width = width or max(1, max(_pages(n, page) for n in lens))
    col = torch.arange(width, device=dev)
    first = need.cumsum(0) - need
    table = order[(first[:, None] + col).clamp_(max=n_pages - 1)].to(torch.int32)
    table = torch.where(col < need[:, None], table, -1).to(torch.int32)
    return table.contiguous(), torch.tensor(lens, device=dev, dtype=torch.int32)


def _normal(shape, dtype, g, fp8=False):
    x = torch.empty(shape, dtype=DTYPES[dtype], device="cuda").normal_(generator=g)
    return x.to(FP8) if fp8 else x


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["kind"] in ("attend", "write"):
        lens = _lengths(c) if c["kind"] == "attend" else [c["T"]] * c["B"]
        n_pages = sum(_pages(n, c["page"]) for n in lens) + 5
        s["table"], s["lens"] = _tables(lens, c["page"], n_pages, g)
        shape = (n_pages, c["page"], c["HKV"], c["D"])
        s["k_cache"], s["v_cache"] = _normal(shape, c["dtype"], g, c["fp8"]), _normal(shape, c["dtype"], g, c["fp8"])
        if c["kind"] == "attend":
            s["q"] = _normal((c["B"], c["H"], c["D"]), c["dtype"], g)
            s["longest"] = max(lens)
        else:
            new = _new_tokens(c)
            s["n"] = sum(new)
            s["offsets"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda") if c["ragged"] else None
            s["k"], s["v"] = _normal((s["n"], c["HKV"], c["D"]), c["dtype"], g), _normal((s["n"], c["HKV"], c["D"]), c["dtype"], g)
        return s
    P = c["page"]
    if c["kind"] == "beam":
        # the beams' tables as a step leaves them: the first beam of a request owns its pages, the others were forked from it
        R, full, begun = c["requests"] * c["beams"], c["T"] // P, c["T"] % P > 0
        mine = c["requests"] * full + (R if begun else 0)
        n_pages, width = mine + 7, full + 2
        order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((c["requests"], c["beams"], width), -1, dtype=torch.int32, device="cuda")
        table[:, :, :full] = order[:c["requests"] * full].view(c["requests"], 1, full)
        counts = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        counts[order[:c["requests"] * full].long()] = c["beams"]
        if begun:
            table[:, :, full] = order[c["requests"] * full:mine].view(c["requests"], c["beams"])
            counts[order[c["requests"] * full:mine].long()] = 1
        table, lens = table.view(R, width), torch.full((R,), c["T"], dtype=torch.int32, device="cuda")
        winner = torch.randint(0, c["beams"], (c["requests"],), generator=g, device="cuda")
        beam = torch.arange(c["beams"], device="cuda")
        losers = torch.argsort((beam == winner[:, None]).to(torch.int8), dim=1, stable=True)[:, :-1]    # all beams but the winner, in order
        base = torch.arange(c["requests"], device="cuda")[:, None] * c["beams"]
        s["children"] = (base + losers).reshape(-1).to(torch.int32)
        s["parents"] = (base + winner[:, None]).expand_as(losers).reshape(-1).to(torch.int32).contiguous()
    elif c["kind"] == "admit":
        # all places taken; the first n sequences have ended and others of the same lengths take their places
        lens_host, n_pages = _spread(c["R"], c["T"]), c["pages"]
        table, lens = _tables(lens_host, P, n_pages, g)
        R, width = table.shape
        valid = torch.arange(width, device="cuda") * P < lens[:, None]
        counts = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        counts[table[valid].long()] = 1
        s["rows"] = torch.randperm(c["n"], generator=g, device="cuda").to(torch.int32)
        s["tokens"] = torch.tensor(lens_host[:c["n"]], dtype=torch.int32, device="cuda")
        s["pages_wanted"] = sum(_pages(n, P) for n in lens_host[:c["n"]])
    else:
        lens_host, kept = _kept(c)
        n_pages = sum(_pages(n, P) for n in lens_host)
        table, _ = _tables(lens_host, P, n_pages, g)
        lens = torch.tensor(kept, dtype=torch.int32, device="cuda")
        R, width = table.shape
        valid = torch.arange(width, device="cuda") * P < lens[:, None]
        counts = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        counts[table[valid].long()] = 1
    layers, HKV, D, dtype = c.get("layers", 1), c.get("HKV", 1), c.get("D", 64), c.get("dtype", "bf16")
    s["caches"] = _normal((layers, 2, n_pages, P, HKV, D), dtype, g)
    s["start"] = torch.cat([counts, lens, table.reshape(-1)])
    if own:
        from hip_attention_b200 import HiPPagePool
        pool = HiPPagePool([x[0] for x in s["caches"]], [x[1] for x in s["caches"]], max_sequences=R, max_pages_per_sequence=width)
        s["pool"], s["state"] = pool, pool.state
    else:
        s["state"] = torch.empty_like(s["start"])
    s["state"].copy_(s["start"])
    s["counts"], s["lens"], s["table"] = s["state"][:n_pages], s["state"][n_pages:n_pages + R], s["state"][n_pages + R:].view(R, width)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _rows_of(cache, slot):
    """Rows of a cache [n_pages, P, HKV, D] in 32 bits."""
    flat = cache.view(-1, *cache.shape[2:])
    if cache.dtype == FP8:
        return flat.view(torch.uint8)[slot].view(FP8).float()
    return flat[slot].float()


def _attend(s):
    c, q = s["case"], s["q"]
    B, P, G = c["B"], c["page"], c["H"] // c["HKV"]
    n = min(c["window"], s["longest"]) if c["window"] else s["longest"]
    t = s["lens"].long()[:, None] - n + torch.arange(n, device=q.device)              # the last n positions of each sequence
    live = t >= 0
    t = torch.where(live, t, 0)
    slot = torch.where(live, s["table"].gather(1, t // P).long() * P + t % P, 0)
    k = _rows_of(s["k_cache"], slot).permute(0, 2, 1, 3)                              # [B, HKV, T, D]
    x = torch.matmul(q.float().view(B, c["HKV"], G, -1), k.transpose(2, 3)) * c["D"] ** -0.5
    del k
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    x = torch.where(live[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    base = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(x - base)
    total = p.sum(-1, keepdim=True)
    v = _rows_of(s["v_cache"], slot).permute(0, 2, 1, 3)
    v = torch.where(live[:, None, :, None], v, 0.0) if c["ragged"] else v
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = (base + torch.log(total)) / math.log(2)
    return out.view(B, c["H"], -1).to(q.dtype), lse.view(B, c["H"])


def _write(s):
    c = s["case"]
    i = torch.arange(s["n"], device="cuda")
    if s["offsets"] is None:
        b, first, count = i // c["n"], i // c["n"] * c["n"], c["n"]
    else:
        b = torch.searchsorted(s["offsets"][1:], i, right=True)
        first, count = s["offsets"][b], s["offsets"][b + 1] - s["offsets"][b]
    t = s["lens"][b] - count + (i - first)
    slot = s["table"][b, t // c["page"]].long() * c["page"] + t % c["page"]
    for new, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
        flat = cache.view(-1, c["HKV"], c["D"])
        if c["fp8"]:
            flat.view(torch.uint8)[slot] = new.float().to(FP8).view(torch.uint8)
        else:
            flat[slot] = new


def _free(s, rows):
    rows = rows.long()
    P = s["case"]["page"]
    pages = s["table"][rows]
    valid = torch.arange(pages.shape[1], device="cuda") * P < s["lens"][rows][:, None]
    s["counts"].index_add_(0, torch.where(valid, pages, 0).reshape(-1).long(), -valid.reshape(-1).to(torch.int32))
    s["lens"][rows] = 0


def _lowest_free(s, n):
    """The n lowest-numbered free pages, ascending."""
    return torch.sort((s["counts"] > 0).to(torch.uint8), stable=True).indices[:n]


def _fork(s, parents, children):
    parents, children, P = parents.long(), children.long(), s["case"]["page"]
    n, lens, pages = parents.numel(), s["lens"][parents], s["table"][parents]
    full, begun = lens // P, lens % P
    shared = torch.arange(pages.shape[1], device="cuda") < full[:, None]
    free, need = _lowest_free(s, n), begun > 0
    place = torch.where(need, need.cumsum(0) - 1, need.sum() + (~need).cumsum(0) - 1)     # (children without a begun page: a free page left as it is)
    to = free[place]
    source = torch.where(need, pages.gather(1, full.long()[:, None].clamp(max=pages.shape[1] - 1))[:, 0].long(), to)
    mine = s["table"][children]
    mine = torch.where(shared, pages, mine)
    at = torch.arange(pages.shape[1], device="cuda") == full[:, None]
    s["table"][children] = torch.where(at & need[:, None], to[:, None].to(torch.int32), mine)
    s["counts"].index_add_(0, torch.where(shared, pages, 0).reshape(-1).long(), shared.reshape(-1).to(torch.int32))
    s["counts"].index_add_(0, to, need.to(torch.int32))
    s["lens"][children] = lens
    copied = (torch.arange(P, device="cuda") < begun[:, None])[:, :, None, None]
    s["caches"][:, :, to] = torch.where(copied, s["caches"][:, :, source], s["caches"][:, :, to])


def _extend(s, rows, tokens):
    rows, P = rows.long(), s["case"]["page"]
    old = s["lens"][rows]
    had, wants = (old + P - 1) // P, (old + tokens + P - 1) // P
    need = (wants - had).long()
    free = _lowest_free(s, s["pages_wanted"])
    entry = torch.repeat_interleave(torch.arange(rows.numel(), device="cuda"), need, output_size=s["pages_wanted"])
    col = had[entry] + torch.arange(s["pages_wanted"], device="cuda") - (need.cumsum(0) - need)[entry]
    s["table"][rows[entry], col] = free.to(torch.int32)
    s["counts"][free] = 1
    s["lens"][rows] = old + tokens


def _compact(s):
    live = s["counts"] > 0
    n = live.sum()
    place = torch.arange(live.numel(), device="cuda")
    to, source = torch.nonzero(~live & (place < n))[:, 0], torch.nonzero(live & (place >= n))[:, 0]
    s["caches"][:, :, to] = s["caches"][:, :, source]
    name = place.to(torch.int32)
    name[source] = to.to(torch.int32)
    valid = torch.arange(s["table"].shape[1], device="cuda") * s["case"]["page"] < s["lens"][:, None]
    s["table"].copy_(torch.where(valid, name[torch.where(valid, s["table"], 0).long()], s["table"]))
    s["counts"][to] = s["counts"][source]
    s["counts"][source] = 0


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _bits(x):
    return x if x.dtype == FP8 else x.view({2: torch.int16, 4: torch.int32}[x.element_size()])


def run(s):
    c = s["case"]
    if c["kind"] == "attend":
        if not own:
            return _attend(s)
        from hip_attention_b200 import paged_decode_attention
        return paged_decode_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], sm_scale=c["D"] ** -0.5,
                                      sliding_window=c["window"] or None, logit_softcap=c["softcap"] or None, return_lse=True)
    if c["kind"] == "write":
        if own:
            from hip_attention_b200 import write_paged_kv
            write_paged_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["lens"], token_offsets=s["offsets"])
        else:
            _write(s)
        return _bits(s["k_cache"]), _bits(s["v_cache"])
    if c["kind"] == "beam":
        if own:
            s["pool"].free(s["children"])
            s["pool"].fork(s["parents"], s["children"])
        else:
            _free(s, s["children"])
            _fork(s, s["parents"], s["children"])
        return _bits(s["caches"]), s["state"]
    if c["kind"] == "admit":
        if own:
            s["pool"].free(s["rows"])
            s["pool"].extend(s["rows"], s["tokens"])
        else:
            _free(s, s["rows"])
            _extend(s, s["rows"], s["tokens"])
        return s["state"]
    s["state"].copy_(s["start"])                # the tables as the sequences that have ended left them
    if own:
        s["pool"].compact()
    else:
        _compact(s)
    return _bits(s["caches"]), s["state"]


# ---------------------------------------------------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(c, seed):
    if c["kind"] not in ("attend", "write"):
        return None                             # whole numbers and copies
    if c["kind"] == "write" and not c["fp8"]:
        return None
    s = prepare(c, seed)
    lens = s["lens"].tolist()

    def sequence(cache, b, lo, hi):
        pages = s["table"][b, lo // c["page"]:-(-hi // c["page"])].long()
        x = cache.view(torch.uint8)[pages].view(FP8) if cache.dtype == FP8 else cache[pages]
        start = lo // c["page"] * c["page"]
        return x.reshape(-1, c["HKV"], c["D"])[lo - start:hi - start].double()

    if c["kind"] == "write":
        new = _new_tokens(c)
        got = []
        for x, cache in ((s["k"], s["k_cache"]), (s["v"], s["v_cache"])):
            flat = cache.double().view(-1, c["HKV"], c["D"])
            at = 0
            for b, n in enumerate(new):
                t = range(lens[b] - n, lens[b])
                page = s["table"][b].tolist()
                slots = torch.tensor([page[j // c["page"]] * c["page"] + j % c["page"] for j in t], device="cuda")
                flat[slots] = x[at:at + n].double()
                at += n
            got.append(flat.view(cache.shape))
        return tuple(got)
    G = c["H"] // c["HKV"]
    out = torch.zeros((c["B"], c["H"], c["D"]), dtype=torch.float64, device="cuda")
    lse = torch.full((c["B"], c["H"]), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        lo = max(0, n - c["window"]) if c["window"] else 0
        if n == 0:
            continue
        k, v = sequence(s["k_cache"], b, lo, n), sequence(s["v_cache"], b, lo, n)
        for h in range(c["H"]):
            x = k[:, h // G] @ s["q"][b, h].double() / math.sqrt(c["D"])
            if c["softcap"]:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            total = torch.logsumexp(x, 0)
            out[b, h] = torch.exp(x - total) @ v[:, h // G]
            lse[b, h] = total / math.log(2)
    return out, lse
