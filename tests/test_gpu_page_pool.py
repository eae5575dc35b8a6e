"""Pages of a pool and writes into them against a model in plain Python: state for state, byte for byte."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e5m2


class Model:
    """Pages are dealt out lowest first, in the order of the entries; a call that cannot be carried out changes nothing."""

    def __init__(self, n_pages, P, R, W, caches):
        self.n, self.P, self.R, self.W = n_pages, P, R, W
        self.refs, self.lens, self.table = [0] * n_pages, [0] * R, [[] for _ in range(R)]
        self.caches = [c.cpu().clone() for c in caches]

    def _pages(self, n):
        return -(-n // self.P)

    def _free_pages(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def extend(self, rows, tokens):
        named = [(r, t) for r, t in zip(rows, tokens) if r >= 0]
        if any(r >= self.R or t < 0 or self._pages(self.lens[r] + t) > self.W for r, t in named) or len({r for r, _ in named}) < len(named):
            return 32
        need = [self._pages(self.lens[r] + t) - self._pages(self.lens[r]) for r, t in named]
        free = self._free_pages()
        if sum(need) > len(free):
            return 16
        for (r, t), k in zip(named, need):
            for _ in range(k):
                page = free.pop(0)
                self.refs[page] = 1
                self.table[r].append(page)
            self.lens[r] += t
        return 0

    def fork(self, parents, children):
        named = [(p, c) for p, c in zip(parents, children) if p >= 0 and c >= 0]
        if any(p >= self.R or c >= self.R or self.lens[c] for p, c in named) or len({c for _, c in named}) < len(named):
            return 32
        free = self._free_pages()
        if sum(self.lens[p] % self.P > 0 for p, _ in named) > len(free):
            return 16
        before = [(self.lens[p], list(self.table[p])) for p, _ in named]
        for (n, pages), (_, c) in zip(before, named):
            full = n // self.P
            self.table[c] = pages[:full]
            for page in pages[:full]:
                self.refs[page] += 1
            if n % self.P:
                page = free.pop(0)
                self.refs[page] = 1
                self.table[c].append(page)
                for x in self.caches:
                    x[page, :n % self.P] = x[pages[full], :n % self.P]
            self.lens[c] = n
        return 0

    def free(self, rows):
        for r in rows:
            if 0 <= r < self.R:
                for page in self.table[r]:
                    self.refs[page] -= 1
                self.table[r], self.lens[r] = [], 0
        return 32 if any(r >= self.R for r in rows) else 0

    def compact(self):
        m = sum(r > 0 for r in self.refs)
        holes = [i for i in range(m) if self.refs[i] == 0]
        movers = [i for i in range(m, self.n) if self.refs[i] > 0]
        for to, src in zip(holes, movers):
            for x in self.caches:
                x[to] = x[src]
            self.refs[to], self.refs[src] = self.refs[src], 0
        name = dict(zip(movers, holes))
        self.table = [[name.get(p, p) for p in pages] for pages in self.table]
        return m


def make(n_pages, P, R, W, layers=2, HKV=2, D=16, dtype=torch.bfloat16, seed=0, layout="plain"):
    from hip_attention_b200 import HiPPagePool
    g = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "plain":
        all_ = [torch.randint(-99, 99, (n_pages, P, HKV, D), generator=g, device="cuda").to(dtype) for _ in range(2 * layers)]
    else:
        both = torch.randint(-99, 99, (layers, n_pages, 2, P, HKV, D), generator=g, device="cuda").to(dtype)
        all_ = [both[i, :, j] for j in range(2) for i in range(layers)]
    pool = HiPPagePool(all_[:layers], all_[layers:], R, W)
    return pool, Model(n_pages, P, R, W, all_), all_


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def same(pool, model, caches, contents=True):
    assert pool.ref_counts.tolist() == model.refs
    assert pool.seq_lens.tolist() == model.lens
    table = pool.block_table.tolist()
    for r, pages in enumerate(model.table):
        assert table[r][:len(pages)] == pages, r
    if contents:
        for x, y in zip(caches, model.caches):
            assert torch.equal(x.cpu().view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("n_pages,P,R,W,layout", [(61, 4, 9, 12, "plain"), (40, 1, 6, 30, "plain"), (500, 16, 33, 40, "interleaved"), (17, 5, 5, 7, "interleaved"), (9000, 2, 20, 900, "plain")])
def test_random_calls_equal_the_model(seed, n_pages, P, R, W, layout):
    """Any calls in any order, among them calls that cannot be carried out."""
    from hip_attention_b200 import read_status
    rng = random.Random(seed)
    pool, model, caches = make(n_pages, P, R, W, seed=seed, layout=layout)
    read_status("cuda")
    kinds = {0: 0, 16: 0, 32: 0}
    for step in range(60):
        do = rng.choice(["extend", "extend", "extend", "fork", "free", "compact"])
        index = rng.choice([torch.int32, torch.int64])
        if do == "extend":
            rows = rng.sample(range(R), rng.randint(1, R)) + [-1] * rng.randint(0, 2)
            rng.shuffle(rows)
            if rng.random() < 0.1:
                rows[0] = rng.choice([R, rows[-1]])
            tokens = [rng.choice([0, 1, 1, rng.randint(0, 2 * P), rng.randint(0, P * W // 2)]) if rng.random() < 0.98 else -1 for _ in rows]
            if rng.random() < 0.2:
                tokens = [1] * len(rows)
                pool.extend(ints(rows, index), 1)
            else:
                pool.extend(ints(rows, index), ints(tokens, index))
            want = model.extend(rows, tokens)
        elif do == "fork":
            empty = [r for r in range(R) if model.lens[r] == 0]
            children = rng.sample(empty, rng.randint(0, len(empty)))
            parents = [rng.randrange(R) for _ in children]
            if rng.random() < 0.2:
                children, parents = children + [-1, rng.randrange(R)], parents + [0, -1]
            if rng.random() < 0.1:
                children, parents = children + [rng.randrange(R)], parents + [rng.randrange(R)]
            if not children:
                continue
            pool.fork(ints(parents, index), ints(children, index))
            want = model.fork(parents, children)
        elif do == "free":
            rows = [rng.randrange(-1, R) for _ in range(rng.randint(1, max(1, R // 2)))]
            if rng.random() < 0.05:
                rows.append(R + 3)
            pool.free(ints(rows, index))
            want = model.free(rows)
        else:
            assert pool.compact().item() == model.compact()
            want = 0
        got = read_status("cuda")
        assert got == want, (step, do)
        kinds[want] += 1
        same(pool, model, caches, contents=do in ("fork", "compact"))
    assert kinds[0] > 20


@pytest.mark.parametrize("P,n_pages", [(1, 70000), (16, 9001)])
def test_large_pools(P, n_pages):
    """More pages than the threads of the plan, sequences longer than a chunk of a table; every page in use once."""
    from hip_attention_b200 import read_status
    R, W = 12, n_pages // 4
    pool, model, caches = make(n_pages, P, R, W, layers=1, HKV=1, D=8)
    read_status("cuda")
    tokens = [W * P, 3 * P + 1, 5, W * P - 1, 0, W * P // 2, 777]
    for rows in (list(range(7)),):
        pool.extend(ints(rows), ints(tokens))
        assert model.extend(rows, tokens) == 0
    pool.fork(ints([0, 3, 6, 0]), ints([7, 8, 9, 10]))
    assert model.fork([0, 3, 6, 0], [7, 8, 9, 10]) == 0
    same(pool, model, caches)
    pool.free(ints([0, 5, 0, 3]))
    model.free([0, 5, 0, 3])
    same(pool, model, caches, contents=False)
    assert pool.compact().item() == model.compact()
    same(pool, model, caches)
    left = model.refs.count(0)
    pool.extend(ints([0]), ints([min(left, W) * P]))          # to the last page
    assert model.extend([0], [min(left, W) * P]) == 0
    same(pool, model, caches, contents=False)
    assert read_status("cuda") == 0


@pytest.mark.parametrize("layers", [1, 65, 140])
def test_layers_beyond_one_launch(layers):
    pool, model, caches = make(12, 4, 4, 6, layers=layers, HKV=1, D=8)
    pool.extend(ints([0, 1]), ints([6, 9]))
    model.extend([0, 1], [6, 9])
    pool.fork(ints([0]), ints([2]))
    model.fork([0], [2])
    pool.free(ints([0]))
    model.free([0])
    same(pool, model, caches)
    pool.compact()
    model.compact()
    same(pool, model, caches)


def test_many_entries():
    R = 4096
    pool, model, caches = make(9000, 2, R, 4, layers=1, HKV=1, D=8)
    rows, tokens = list(range(R))[::-1], [i % 5 for i in range(R)]
    pool.extend(ints(rows), ints(tokens))
    assert model.extend(rows, tokens) == 0
    same(pool, model, caches, contents=False)
    pool.free(ints(rows[:2000] + rows[:2000]))
    model.free(rows[:2000])
    parents = [rows[3000 + i % 1000] for i in range(2000)]
    pool.fork(ints(parents), ints(rows[:2000]))
    assert model.fork(parents, rows[:2000]) == 0
    same(pool, model, caches)
    pool.free(ints(rows))
    model.free(rows)
    assert pool.compact().item() == 0
    same(pool, model, caches)


def test_state_is_one_buffer():
    """A checkpoint is one copy: calls after it has been put back go as they went before."""
    pool, model, caches = make(40, 4, 6, 8)
    pool.extend(ints([0, 3]), ints([9, 17]))
    saved = pool.state.clone()
    pool.extend(ints([1]), 5)
    first = pool.state.clone()
    pool.state.copy_(saved)
    pool.extend(ints([1]), 5)
    assert torch.equal(pool.state, first)


def test_refusals_of_pools_and_entries():
    from hip_attention_b200 import HiPPagePool
    c = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t, device="cuda")   # noqa: E731
    for k, v, R, W in (([c(4, 4, 2, 16)], [c(4, 4, 2, 16), c(4, 4, 2, 16)], 2, 2), ([c(4, 4, 2, 16)], [c(4, 4, 2, 8)], 2, 2), ([c(4, 4, 2, 16)], [c(4, 4, 2, 16).half()], 2, 2),
                       ([c(4, 4, 1, 4)], [c(4, 4, 1, 4)], 2, 2), ([c(4, 2, 4, 16).transpose(1, 2)], [c(4, 2, 4, 16).transpose(1, 2)], 2, 2),
                       ([c(4, 4, 2, 16)], [c(4, 4, 2, 16)], 0, 2), ([c(4, 4, 2, 16)], [c(4, 4, 2, 16)], 2, 0), ([c(4, 4, 2, 16)], [c(4, 4, 2, 16)], 262145, 2),
                       ([c(4, 4, 2, 16, t=torch.int64)], [c(4, 4, 2, 16, t=torch.int64)], 2, 2), ([c(4, 4, 2, 16).cpu()], [c(4, 4, 2, 16)], 2, 2)):
        with pytest.raises(ValueError):
            HiPPagePool(k, v, R, W)
    pool, _, _ = make(8, 4, 3, 4)
    for bad in (lambda: pool.extend(ints([0]).float(), 1), lambda: pool.extend(ints([0]), ints([1, 2])), lambda: pool.extend(ints([0]), -1), lambda: pool.extend(ints([0]).cpu(), 1),
                lambda: pool.extend(ints([[0]]), 1), lambda: pool.fork(ints([0, 1]), ints([2])), lambda: pool.free(torch.zeros(5000, dtype=torch.int32, device="cuda")),
                lambda: pool.free(ints([0, 1, 2, 0])[::2])):
        with pytest.raises(ValueError):
            bad()
    before = pool.state.clone()
    pool.extend(ints([]), 1)
    pool.fork(ints([]), ints([]))
    pool.free(ints([]))
    pool.free(ints([2 ** 40, -2 ** 40], torch.int64))
    assert torch.equal(pool.state, before)


# ---------------------------------------------------------------------------------------------------------------------
# writes
# ---------------------------------------------------------------------------------------------------------------------
def _pool(n_pages, P, HKV, D, cache_type, g):
    c = torch.randn((n_pages, P, HKV, D), generator=g, device="cuda")
    return c.to(cache_type)


def _bits(x):
    return x.contiguous().view(torch.uint8)


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32), (torch.bfloat16, FP8),
                                         (torch.float16, FP8), (torch.bfloat16, torch.uint8)])
@pytest.mark.parametrize("P,HKV,D", [(1, 2, 64), (16, 8, 128), (20, 1, 8), (64, 3, 40)])
def test_writes(dtype, cache, P, HKV, D):
    from hip_attention_b200 import read_status, write_paged_kv
    g = torch.Generator(device="cuda").manual_seed(P)
    R, W = 6, -(-200 // P)
    n_pages = R * W + 2
    ct = FP8 if cache == torch.uint8 else cache
    kc, vc = _pool(n_pages, P, HKV, D, ct, g), _pool(n_pages, P, HKV, D, ct, g)
    view = (lambda c: c.view(torch.uint8)) if cache == torch.uint8 else (lambda c: c)
    table = torch.randperm(n_pages, generator=g, device="cuda")[:R * W].view(R, W)
    read_status("cuda")
    for index, rows, lens, new in ((torch.int32, None, [200, 1, 33, 64, 17, 2], [70, 1, 0, 64, 16, 1]), (torch.int64, [4, -1, 0, 2], [200, 1, 33, 64, 17, 2], [17, 5, 3, 33]),
                                   (torch.int32, None, [200, 1, 33, 64, 17, 2], None)):
        new_ = new or [1] * R
        n = sum(new_)
        more = 3 if new else 0          # (rows behind the last sequence)
        k, v = (torch.randn((n + more, HKV, D), generator=g, device="cuda").to(dtype) * 3 for _ in range(2))
        offs = torch.tensor([sum(new_[:i]) for i in range(len(new_) + 1)], dtype=index, device="cuda") if new else None
        want = [kc.view(torch.uint8 if ct == FP8 else ct).clone(), vc.view(torch.uint8 if ct == FP8 else ct).clone()]
        at = 0
        for b, m in enumerate(new_):
            r = rows[b] if rows else b
            for j in range(m):
                if r >= 0:
                    t = lens[r] - m + j
                    for x, w in ((k, want[0]), (v, want[1])):
                        y = x[at].to(ct)
                        w[int(table[r, t // P]), t % P] = y.view(torch.uint8) if ct == FP8 else y
                at += 1
        write_paged_kv(k, v, view(kc), view(vc), table.to(index), torch.tensor(lens, dtype=index, device="cuda"),
                       rows=torch.tensor(rows, dtype=index, device="cuda") if rows else None, token_offsets=offs)
        assert torch.equal(_bits(kc), _bits(want[0])) and torch.equal(_bits(vc), _bits(want[1]))
    assert read_status("cuda") == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_16_bit_value_to_fp8(dtype):
    """All 65536 values: nearest e5m2, ties to even, infinities beyond the range; NaN stays NaN."""
    from hip_attention_b200 import write_paged_kv
    x = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype).view(64, 8, 128)
    kc, vc = (torch.zeros((4, 16, 8, 128), dtype=FP8, device="cuda") for _ in range(2))
    write_paged_kv(x, x, kc, vc, ints([[2, 0, 3, 1]]), ints([64]))
    got, want = kc[[2, 0, 3, 1]].view(64, 8, 128).double(), x.float().to(FP8).double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(1e9), want.nan_to_num(1e9))


def test_strided_tokens_and_heads_first_pools():
    from hip_attention_b200 import write_paged_kv
    g = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.randn((5, 12, 64), generator=g, device="cuda").to(torch.bfloat16)     # queries, keys and values of a fused projection
    kc, vc = (torch.zeros((3, 2, 4, 64), dtype=torch.bfloat16, device="cuda").transpose(1, 2) for _ in range(2))
    write_paged_kv(qkv[:, 8:10], qkv[:, 10:12], kc, vc, ints([[1, 2]]), ints([7]))
    flat = torch.cat([kc[1], kc[2]])
    assert torch.equal(flat[2:7], qkv[:, 8:10]) and not flat[:2].any() and not flat[7:].any() and not kc[0].any()
    assert torch.equal(torch.cat([vc[1], vc[2]])[2:7], qkv[:, 10:12])


def test_writes_out_of_range_are_left_out():
    from hip_attention_b200 import _lib as L, read_status, write_paged_kv
    kc, vc = (torch.zeros((3, 4, 1, 8), dtype=torch.float32, device="cuda") for _ in range(2))
    k = torch.ones((4, 1, 8), device="cuda")
    read_status("cuda")
    for table, lens, rows, bit in (([[0, 1]], [2], None, L.STATUS_TOKEN_RANGE), ([[0, 1]], [9], None, L.STATUS_TOKEN_RANGE), ([[0, 3]], [6], None, L.STATUS_PAGE_RANGE),
                                   ([[0, -1]], [6], None, L.STATUS_PAGE_RANGE), ([[0, 1]], [4], [1], L.STATUS_SEQUENCE)):
        kc.zero_()
        write_paged_kv(k, k, kc, vc, ints(table), ints(lens), rows=ints(rows) if rows else None)
        assert read_status("cuda") == bit
        assert kc.sum().item() == 8 * {2: 2, 9: 3, 6: 2, 4: 0}[lens[0]]
    for bad in (lambda: write_paged_kv(k, k, kc, vc, ints([[0, 1], [1, 2], [0, 2]]), ints([4, 4, 4])), lambda: write_paged_kv(k.half(), k.half(), kc, vc, ints([[0]]), ints([4])),
                lambda: write_paged_kv(k, k[:3], kc, vc, ints([[0]]), ints([4])), lambda: write_paged_kv(k, k, kc, vc, ints([[0]]), ints([4]), token_offsets=ints([0])),
                lambda: write_paged_kv(k[..., :4], k[..., :4], kc, vc, ints([[0]]), ints([4])), lambda: write_paged_kv(k.cpu(), k, kc, vc, ints([[0]]), ints([4]))):
        with pytest.raises(ValueError):
            bad()
    write_paged_kv(k[:0], k[:0], kc, vc, ints([[0]]), ints([4]))
