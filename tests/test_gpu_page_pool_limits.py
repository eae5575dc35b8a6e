"""A page pool at the limits that its calls document: the longest sequences, pages of many tokens, pools dropped or out of pages while they are used."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("P", [65537, 70000, 2 ** 31 - 1])
def test_the_longest_sequence_in_pages_of_many_tokens(P):
    """length + page_size - 1 passes 2^31: page counts are made in 64 bits."""
    from hip_attention_b200 import _lib as L, read_status
    from hip_attention_b200.operator import status_word
    lib, st = L.load(), torch.cuda.current_stream().cuda_stream
    longest = 0x7fff0000
    need = -(-longest // P)
    n_pages, R, W = 2 * need + 5, 3, need + 1
    refs, lens, table = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((n_pages,), (R,), (R, W)))
    p = L.PagePool(ref_counts=refs.data_ptr(), seq_lens=lens.data_ptr(), block_table=table.data_ptr(), status=status_word("cuda").data_ptr(), n_pages=n_pages, page_size=P,
                   n_sequences=R, table_width=W)
    read_status("cuda")

    def extend(rows, tokens):
        a, b = ints(rows), ints(tokens)
        L.check(lib.hipattn_pool_extend(C.byref(p), a.data_ptr(), b.data_ptr(), 0, len(rows), st), "extend")
        return read_status("cuda")

    assert extend([1, 0], [longest - 1, 5]) == 0
    assert lens.tolist() == [5, longest - 1, 0] and table[1, :need].tolist() == list(range(need)) and table[0, 0].item() == need
    assert int(refs.sum()) == need + 1 and int(refs[:need + 1].min()) == 1
    assert extend([1], [1]) == 0 and lens.tolist() == [5, longest, 0] and int(refs.sum()) == need + 1      # to the last token
    assert extend([1], [1]) == L.STATUS_SEQUENCE and extend([0], [2 ** 31 - 1]) == L.STATUS_SEQUENCE
    assert lens.tolist() == [5, longest, 0] and int(refs.sum()) == need + 1
    a = ints([1])
    L.check(lib.hipattn_pool_free(C.byref(p), a.data_ptr(), 1, st), "free")
    assert read_status("cuda") == 0 and lens.tolist() == [5, 0, 0] and refs[need].item() == 1 and int(refs.sum()) == 1


def _bits(pool):
    return [c.view(torch.int16).clone() for c in pool.k_caches + pool.v_caches] + [pool.state.clone()]


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("n_tokens", ["int", "tensor"])
def test_a_step_of_a_pool_that_runs_out_writes_nothing(captured, n_tokens):
    """A growth that is refused names no rows, so the writes behind it leave the last tokens as they were, one of them in a page that
    two sequences share; a graph of the step goes on when there are pages again."""
    from hip_attention_b200 import HiPPagePool, paged_decode_attention, read_status, write_paged_kv
    P, HKV, D, layers = 4, 2, 64, 2
    g = torch.Generator(device="cuda").manual_seed(0)
    caches = [torch.randn((5, P, HKV, D), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2 * layers)]
    pool = HiPPagePool(caches[:layers], caches[layers:], 4, 6)
    k, v, q = (torch.randn((4, n, D), generator=g, device="cuda").to(torch.bfloat16) for n in (HKV, HKV, 4))
    rows, one = ints([0, 1, -1, 2]), ints([1, 1, 1, 1])
    out = torch.full((layers, 4, 4, D), 7.0, dtype=torch.bfloat16, device="cuda")
    pool.extend(ints([0, 1]), ints([2 * P, P - 1]))        # pages 0 to 2
    pool.fork(ints([0]), ints([2]))                        # two full pages shared; two pages are free, a step needs two, then none
    read_status("cuda")

    def step():
        pool.extend(rows, one if n_tokens == "tensor" else 1, grown)
        for l in range(layers):
            write_paged_kv(k, v, pool.k_caches[l], pool.v_caches[l], pool.block_table, pool.seq_lens, rows=grown)
            paged_decode_attention(q, pool.k_caches[l], pool.v_caches[l], pool.block_table, pool.seq_lens, rows=grown, out=out[l])
        return grown
    grown = torch.zeros_like(rows)
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        run = lambda: (graph.replay(), grown)[1]   # noqa: E731
    else:
        run = step
    pool.extend(ints([3]), 2 * P)                          # the last two pages
    assert read_status("cuda") == 0
    before = _bits(pool)
    assert run().tolist() == [-1, -1, -1, -1] and read_status("cuda") == 16
    assert all(torch.equal(a, b) for a, b in zip(before, _bits(pool))) and not out.any()
    pool.free(ints([3]))
    assert run().tolist() == [0, 1, -1, 2] and read_status("cuda") == 0
    lens = pool.seq_lens.tolist()
    assert lens == [2 * P + 1, P, 2 * P + 1, 0]
    for l in range(layers):
        for i, r in ((0, 0), (1, 1), (3, 2)):
            page, at = pool.block_table[r, (lens[r] - 1) // P], (lens[r] - 1) % P
            assert torch.equal(pool.k_caches[l][page, at], k[i]) and torch.equal(pool.v_caches[l][page, at], v[i])
        assert torch.equal(pool.k_caches[l][:2].view(torch.int16), before[l][:2])       # the shared pages
    assert out[:, [0, 1, 3]].any(-1).all() and not out[:, 2].any()


def test_rows_that_grew():
    """-1 for entries that are left out and for every entry of a call that is refused, whatever the reason; `rows` itself may receive them."""
    from hip_attention_b200 import HiPPagePool, read_status
    c = [torch.zeros((9000, 2, 1, 8), dtype=torch.float16, device="cuda") for _ in range(2)]
    for n_pages in (12, 9000):            # planned by one CTA, and by a cluster
        pool = HiPPagePool([c[0][:n_pages]], [c[1][:n_pages]], 5, 9)
        read_status("cuda")

        def grow(rows, tokens):
            grown = torch.full((len(rows),), 99, dtype=torch.int32, device="cuda")
            assert pool.extend(ints(rows), tokens, grown) is grown
            return grown.tolist()
        grown = torch.empty(4, dtype=torch.int32, device="cuda")
        pool.extend(torch.tensor([3, -1, 0, -7], device="cuda"), ints([3, 5, 0, 1]), grown)
        assert grown.tolist() == [3, -1, 0, -1] and read_status("cuda") == 0
        for rows, tokens in (([0, 0], [1, 1]), ([0, 5], [1, 1]), ([0, 1], [1, -1]), ([0, 1], [1, 19])):
            assert grow(rows, ints(tokens)) == [-1, -1] and read_status("cuda") == 32
        if n_pages == 12:
            assert grow([0, 1, 2], 8) == [-1, -1, -1] and read_status("cuda") == 16
        assert grow([], 1) == [] and pool.extend(ints([0]), 0) is None
        rows = ints([4, -2])
        pool.extend(rows, 1, rows)
        assert rows.tolist() == [4, -1] and pool.seq_lens.tolist() == [0, 0, 0, 3, 1]
        for bad in (torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(2, dtype=torch.int64, device="cuda"), torch.empty(2, dtype=torch.int32),
                    torch.empty(4, dtype=torch.int32, device="cuda")[::2]):
            with pytest.raises(ValueError, match="grown"):
                pool.extend(ints([0, 1]), 1, bad)
        assert pool.seq_lens.tolist() == [0, 0, 0, 3, 1] and read_status("cuda") == 0


def test_a_pool_dropped_while_its_calls_run_on_another_stream():
    """What the pool allocated is not given to others before the stream that uses it has passed, and the calls end as they should."""
    from hip_attention_b200 import HiPPagePool, read_status
    n_pages, P, R, W = 300, 4, 40, 50
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn((n_pages, P, 1, 16), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    pool = HiPPagePool([k], [v], R, W)
    pool.extend(ints([1, 0]), ints([8 * P, 6 * P + 3]))       # pages 0 to 7, 8 to 14
    pool.free(ints([1]))
    parents, children = ints([0]), ints([2])
    k0, v0 = k.clone(), v.clone()
    read_status("cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    sizes = [pool.state.numel() * 4, 4096 * 12 + 16]
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)
        pool.fork(parents, children)          # page 14's three tokens to page 0
        pool.compact()                        # eight pages: 0, 8 .. 14; 8 .. 14 to 1 .. 7
    del pool
    others = [torch.zeros(n, dtype=torch.uint8, device="cuda") for n in sizes * 30]
    assert not side.query()                   # (the calls have not begun)
    torch.cuda.synchronize()
    assert not any(bool(x.any()) for x in others) and read_status("cuda") == 0
    for c, c0 in ((k, k0), (v, v0)):
        assert torch.equal(c[1:8], c0[8:15]) and torch.equal(c[0, :3], c0[14, :3]) and torch.equal(c[0, 3], c0[0, 3]) and torch.equal(c[8:], c0[8:])


def test_sizes_beyond_32_bits_are_refused():
    """Sizes whose lower 32 bits alone would look ordinary (expanded tensors: nothing of that size is there)."""
    from hip_attention_b200 import HiPPagePool, paged_decode_attention, write_paged_kv
    big = 2 ** 32 + 4
    c = torch.zeros((4, 4, 2, 64), dtype=torch.bfloat16, device="cuda")
    pages, tokens = c[:1].expand(big, 4, 2, 64), c[:, :1].expand(4, big, 2, 64)
    q, table, lens = torch.zeros((1, 4, 64), dtype=torch.bfloat16, device="cuda"), ints([[0, 1]]), ints([3])
    k = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device="cuda")
    many = q.expand(big, 4, 64)
    for bad in (lambda: paged_decode_attention(q, pages, pages, table, lens), lambda: paged_decode_attention(q, tokens, tokens, table, lens),
                lambda: paged_decode_attention(many, c, c, table, lens), lambda: write_paged_kv(k, k, pages, pages, table, lens),
                lambda: write_paged_kv(k, k, tokens, tokens, table, lens), lambda: paged_decode_attention(q, c, c, table.expand(big, 2), lens),
                lambda: HiPPagePool([tokens], [tokens], 2, 2)):
        with pytest.raises(ValueError, match="2\\^31"):
            bad()
    with pytest.raises(ValueError, match="at most"):
        HiPPagePool([pages], [pages], 2, 2)


def test_expanded_tensors_are_not_written_to():
    """They may be read: a cache of one page seen as many."""
    from hip_attention_b200 import paged_decode_attention, write_paged_kv
    c = torch.randn((4, 4, 2, 64), device="cuda").to(torch.bfloat16)
    q, table, lens = torch.ones((2, 4, 64), dtype=torch.bfloat16, device="cuda"), ints([[0, 1], [2, 3]]), ints([3, 8])
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    same = c[:1].expand(4, 4, 2, 64)
    for bad in (lambda: paged_decode_attention(q, c, c, table, lens, out=q[:1].expand(2, 4, 64)), lambda: write_paged_kv(k, k, same, c, table, lens),
                lambda: write_paged_kv(k, k, c, c[:, :, :1].expand(4, 4, 2, 64), table, lens)):
        with pytest.raises(ValueError, match="share memory"):
            bad()
    got = paged_decode_attention(q, same, same, table, lens)
    assert torch.equal(got, paged_decode_attention(q, same.contiguous(), same.contiguous(), table, lens))
    assert torch.equal(got, paged_decode_attention(q, c, c, torch.zeros_like(table), lens))
