"""The page pool's operators together, as a serving loop runs them, and next to the package's sparse attention on the same pool."""
import random

import pytest
import torch

from test_gpu_paged_attention import DT, check, reference

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e5m2


class Server:
    """A toy serving loop over a pool; it keeps every sequence's keys and values itself, in 64 bits, to compare with."""

    def __init__(self, layers, n_pages, P, R, W, HKV, D, dtype, fp8=False, seed=0):
        from hip_attention_b200 import HiPPagePool
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype, self.cache_type, self.HKV, self.D, self.R = DT[dtype], FP8 if fp8 else DT[dtype], HKV, D, R
        make = lambda: torch.full((n_pages, P, HKV, D), float("nan"), device="cuda").to(self.cache_type)   # noqa: E731
        self.pool = HiPPagePool([make() for _ in range(layers)], [make() for _ in range(layers)], R, W)
        self.kept = [[[torch.zeros((0, HKV, D), dtype=torch.float64, device="cuda") for _ in range(2)] for _ in range(layers)] for _ in range(R)]

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def append(self, rows, counts):
        """Grows the sequences and writes their new tokens in all layers."""
        from hip_attention_b200 import write_paged_kv
        self.pool.extend(self.ints(rows), self.ints(counts))
        offsets = self.ints([sum(counts[:i]) for i in range(len(counts) + 1)])
        for l, (kc, vc) in enumerate(zip(self.pool.k_caches, self.pool.v_caches)):
            k, v = (torch.randn((sum(counts), self.HKV, self.D), generator=self.g, device="cuda").to(self.dtype) for _ in range(2))
            write_paged_kv(k, v, kc, vc, self.pool.block_table, self.pool.seq_lens, rows=self.ints(rows), token_offsets=offsets)
            at = 0
            for r, n in zip(rows, counts):
                for i, x in enumerate((k, v)):
                    if r >= 0:
                        self.kept[r][l][i] = torch.cat([self.kept[r][l][i], x[at:at + n].to(self.cache_type).double()])
                at += n

    def attend(self, rows, H, **kw):
        from hip_attention_b200 import paged_decode_attention
        scale = self.D ** -0.5
        none = torch.zeros((0, self.HKV, self.D), dtype=torch.float64, device="cuda")
        for l, (kc, vc) in enumerate(zip(self.pool.k_caches, self.pool.v_caches)):
            q = torch.randn((len(rows), H, self.D), generator=self.g, device="cuda").to(self.dtype)
            out, lse = paged_decode_attention(q, kc, vc, self.pool.block_table, self.pool.seq_lens, rows=self.ints(rows), sm_scale=scale, return_lse=True, **kw)
            keys, vals = ([self.kept[r][l][i] if r >= 0 else none for r in rows] for i in range(2))
            check(out, lse, reference(q, keys, vals, scale, kw.get("sliding_window"), kw.get("logit_softcap"), self.dtype != torch.float32), q.dtype)


@pytest.mark.parametrize("dtype,fp8,P", [("bf16", False, 16), ("fp16", True, 1), ("fp32", False, 5), ("bf16", True, 64)])
def test_a_serving_loop(dtype, fp8, P):
    """Prompts, steps of new tokens, beams forked from one another, ended sequences, a compaction: attention is right after each."""
    from hip_attention_b200 import read_status
    rng = random.Random(P)
    s = Server(2, 6000 // P + 60, P, 12, 900 // P + 2, 2, 64, dtype, fp8, seed=P)
    read_status("cuda")
    s.append([0, 1, 2, 5], [130, 1, 3 * P, 77])
    s.attend([0, 1, 2, 5, -1], 8)
    s.pool.fork(s.ints([0, 0, 2]), s.ints([3, 4, 6]))
    for parent, child in ((0, 3), (0, 4), (2, 6)):
        s.kept[child] = [[x for x in pair] for pair in s.kept[parent]]
    s.attend(list(range(7)), 8)
    for step in range(6):
        s.append([0, 1, 2, 3, 4, 5, 6, -1], [1] * 8)           # a padded batch
        s.attend([6, 5, 4, 3, 2, 1, 0, -1], 8, sliding_window=[None, 50][step & 1])
    s.pool.free(s.ints([0, 5, -1, 0]))
    for r in (0, 5):
        s.kept[r] = [[x[:0] for x in pair] for pair in s.kept[r]]
    s.attend(list(range(7)), 8)
    s.append([5, 9, 11], [rng.randint(1, 300) for _ in range(3)])
    used = s.pool.compact()
    assert used.item() == int((s.pool.ref_counts > 0).sum()) and bool((s.pool.ref_counts[used.item():] == 0).all())
    s.append([1, 3, 9], [P, 1, 2 * P + 1])
    s.attend([9, 3, 1, 11, 6, 0], 8, logit_softcap=20.0)
    assert read_status("cuda") == 0


@pytest.mark.parametrize("P", [1, 16])
def test_next_to_the_sparse_operator(P):
    """With sink and window over the whole sequence hip_attention_12 attends what the exact operator does, through the same pool, table and
    lengths; two 16-bit results of the same numbers."""
    from hip_attention_b200 import HiPAttentionArgs, ScanStage, hip_attention_12, paged_decode_attention
    s = Server(1, 3000 // P + 50, P, 4, 1024 // P, 2, 128, "bf16", seed=3)
    s.append([0, 1, 2, 3], [600, 33, 257, 900])
    s.attend([0, 1, 2, 3], 8)
    q = torch.randn((4, 8, 128), generator=s.g, device="cuda").to(torch.bfloat16) * 128 ** -0.5
    exact = paged_decode_attention(q, s.pool.k_caches[0], s.pool.v_caches[0], s.pool.block_table, s.pool.seq_lens)
    args = HiPAttentionArgs(position_ids=(s.pool.seq_lens.long() - 1)[:, None], sink_token_size=64, sliding_window_size=960, second_stage_k=64, block_size_k=64,
                            stages=[ScanStage(64, 1, 32, None, 1), ScanStage(64, 1, 8, 64, 1)], block_sparse_block_size_q=64, model_context_length=1024,
                            extend_context_length=1024, k_cache=s.pool.k_caches[0], v_cache=s.pool.v_caches[0], block_table=s.pool.block_table, cache_seq_lens=s.pool.seq_lens)
    sparse, _ = hip_attention_12(q[:, None], None, None, args=args)
    # the sparse kernel's weights have one 16-bit term (2^-9 of each): both outputs are roundings of sums that differ by at most 2^-8 of sum p |v| < 4
    assert (sparse[:, 0].float() - exact.float()).abs().max().item() <= 2 * 2.0 ** -8 * 4


def test_a_captured_step_replayed():
    """One graph of a whole step (grow, write, attend), replayed with other rows, among them fewer than it was captured with."""
    from hip_attention_b200 import paged_decode_attention, read_status, write_paged_kv
    P, R, H, HKV, D = 4, 6, 4, 2, 64
    runs = []
    for captured in (False, True):
        s = Server(1, 80, P, R, 20, HKV, D, "bf16", seed=1)
        s.append([0, 1, 2], [5, 8, 3])
        rows = s.ints([0, 1, 2, -1])
        k, v, q = (torch.zeros((4, n, D), dtype=torch.bfloat16, device="cuda") for n in (HKV, HKV, H))
        out = torch.empty_like(q)

        def step():
            s.pool.extend(rows, 1)
            write_paged_kv(k, v, s.pool.k_caches[0], s.pool.v_caches[0], s.pool.block_table, s.pool.seq_lens, rows=rows)
            paged_decode_attention(q, s.pool.k_caches[0], s.pool.v_caches[0], s.pool.block_table, s.pool.seq_lens, rows=rows, out=out)
        run = step
        if captured:
            saved = s.pool.state.clone()
            graph = torch.cuda.CUDAGraph()
            side = torch.cuda.Stream()
            with torch.cuda.graph(graph, stream=side):
                step()
            s.pool.state.copy_(saved)
            run = graph.replay
        g, outs = torch.Generator(device="cuda").manual_seed(9), []
        for i in range(12):
            rows.copy_(s.ints([[0, 1, 2, -1], [0, -1, 2, 4], [-1, -1, -1, -1], [4, 1, 0, 2]][i % 4]))
            for x in (k, v, q):
                x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            run()
            outs.append(out.clone())
        runs.append((outs, s.pool.state.clone()))
    torch.cuda.synchronize()
    assert read_status("cuda") == 0
    assert all(torch.equal(a, b) for a, b in zip(runs[0][0], runs[1][0])) and torch.equal(runs[0][1], runs[1][1])


def test_captured_pool_calls_replayed():
    """Two graphs of one pool's calls alive at once: each replay works on the pool as the calls before left it."""
    from hip_attention_b200 import read_status
    results = []
    for captured in (False, True):
        s = Server(2, 64, 4, 8, 12, 1, 16, "fp16", seed=2)
        s.append([0, 1], [9, 14])
        a, b = s.ints([0, 1]), s.ints([2, 3])

        def beam():
            s.pool.free(b)
            s.pool.fork(a, b)

        def tidy():
            s.pool.free(a[:1])
            s.pool.compact()
            s.pool.extend(a[:1], 7)
        fs = [beam, tidy]
        if captured:
            saved = s.pool.state.clone(), [c.clone() for c in s.pool.k_caches]
            graphs = [torch.cuda.CUDAGraph() for _ in fs]
            for gr, f in zip(graphs, fs):
                with torch.cuda.graph(gr):
                    f()
            fs = [gr.replay for gr in graphs]
            assert torch.equal(saved[0], s.pool.state)
        for i in (0, 0, 1, 0, 1, 1, 0):
            fs[i]()
        torch.cuda.synchronize()
        results.append([s.pool.state.clone()] + [c.view(torch.int16).clone() for c in s.pool.k_caches])
    assert read_status("cuda") == 0
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_on_a_stream_of_its_own():
    s = Server(1, 200, 16, 4, 40, 2, 64, "bf16", seed=4)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        s.append([0, 2], [300, 41])
        s.pool.fork(s.ints([2]), s.ints([1]))
        s.kept[1] = [[x for x in pair] for pair in s.kept[2]]
        s.pool.compact()
        s.append([1], [9])
        s.attend([0, 1, 2, 3], 4)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()


def test_calls_of_the_c_interface():
    """The pool's calls through the C interface give what the Python names give."""
    import ctypes as C
    from hip_attention_b200 import _lib as L, paged_decode_attention
    from hip_attention_b200.operator import _tokens, status_word
    lib, status, st = L.load(), status_word("cuda").data_ptr(), torch.cuda.current_stream().cuda_stream
    R, W, P, n_pages, HKV, D = 5, 300, 4, 1500, 2, 64
    kc, vc = (torch.zeros((n_pages, P, HKV, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    refs, lens, table = (torch.zeros(s, dtype=torch.int32, device="cuda") for s in ((n_pages,), (R,), (R, W)))
    caches = (C.c_void_p * 2)(kc.data_ptr(), vc.data_ptr())
    p = L.PagePool(ref_counts=refs.data_ptr(), seq_lens=lens.data_ptr(), block_table=table.data_ptr(), caches=C.cast(caches, C.POINTER(C.c_void_p)),
                   page_stride=P * HKV * D * 2, page_bytes=P * HKV * D * 2, status=status, n_pages=n_pages, page_size=P, n_sequences=R, table_width=W, n_caches=2)
    scratch = torch.empty(max(lib.hipattn_pool_scratch(C.byref(p), 8), lib.hipattn_pool_scratch(C.byref(p), 0)), dtype=torch.uint8, device="cuda")
    p.scratch = scratch.data_ptr()
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    rows, new = ints([0, 3]), ints([1111, 6])
    L.check(lib.hipattn_pool_extend(C.byref(p), rows.data_ptr(), new.data_ptr(), 0, 2, st), "extend")
    k, v = (torch.randn((1117, HKV, D), device="cuda").to(torch.bfloat16) for _ in range(2))
    off = ints([0, 1111, 1117])
    w = L.WriteKvParams(k=k.data_ptr(), v=v.data_ptr(), k_stride_t=HKV * D, k_stride_h=D, v_stride_t=HKV * D, v_stride_h=D, k_pool=_tokens(None, kc, table, lens, "k"),
                        v_pool=_tokens(None, vc, table, lens, "v"), rows=rows.data_ptr(), offsets=off.data_ptr(), status=status, N=1117, dtype=L.BF16, D=D, B=2, HKV=HKV, n_rows=R)
    L.check(lib.hipattn_write_kv(C.byref(w), st), "write")
    a, b = ints([3, 0]), ints([1, 4])
    L.check(lib.hipattn_pool_fork(C.byref(p), a.data_ptr(), b.data_ptr(), 2, st), "fork")
    L.check(lib.hipattn_pool_free(C.byref(p), a.data_ptr(), 1, st), "free")
    used = ints([0])
    L.check(lib.hipattn_pool_compact(C.byref(p), used.data_ptr(), st), "compact")
    assert used.item() == int((refs > 0).sum()) and lens.tolist() == [1111, 6, 0, 0, 1111]
    q = torch.randn((R, 4, D), device="cuda").to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty((R, 4), device="cuda")
    d = L.PagedDecodeParams(q=q.data_ptr(), q_stride_b=4 * D, q_stride_h=D, out=out.data_ptr(), o_stride_b=4 * D, o_stride_h=D, lse_out=lse.data_ptr(),
                            k=_tokens(None, kc, table, lens, "k"), v=_tokens(None, vc, table, lens, "v"), status=status, dtype=L.BF16, D=D, B=R, H=4, HKV=HKV, n_rows=R, sm_scale=0.2)
    room = torch.empty(max(16, lib.hipattn_paged_decode_scratch(C.byref(d))), dtype=torch.uint8, device="cuda")
    d.scratch, d.scratch_bytes = room.data_ptr(), room.numel()
    L.check(lib.hipattn_paged_decode(C.byref(d), st), "decode")
    want, want_lse = paged_decode_attention(q, kc, vc, table, lens, sm_scale=0.2, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    keys = [k[:1111].double(), k[1111:].double()]
    vals = [v[:1111].double(), v[1111:].double()]
    none = torch.zeros((0, HKV, D), dtype=torch.float64, device="cuda")
    check(out, lse, reference(q, [keys[0], keys[1], none, none, keys[0]], [vals[0], vals[1], none, none, vals[0]], 0.2), q.dtype)


def test_first_call_of_a_process_captured():
    """A process whose first call is captured: the status word is not part of the graph, neither its memory nor its zeros."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = """
import torch
from hip_attention_b200 import paged_decode_attention, read_status
kc, vc = (torch.randn((4, 4, 2, 64), device='cuda') for _ in range(2))
q, table, lens = torch.randn((1, 4, 64), device='cuda'), torch.tensor([[2, 9]], device='cuda'), torch.tensor([3], device='cuda')
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = paged_decode_attention(q, kc, vc, table, lens)
graph.replay()
assert read_status('cuda') == 0
want = paged_decode_attention(q, kc, vc, table, lens)
assert torch.equal(out, want)
lens.fill_(6)                      # the second page is out of range
graph.replay()
assert read_status('cuda') == 1 and read_status('cuda') == 0
del out, graph
torch.cuda.empty_cache()
lens.fill_(3)
assert torch.equal(paged_decode_attention(q, kc, vc, table, lens), want) and read_status('cuda') == 0
print('fine')
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("width,n", [(64, 900), (4096, 900)])
def test_first_launch_of_a_kernel_captured(width, n):
    """The first call that joins parts (in a cluster; over shares, with a second launch) may be a captured one."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = f"""
import torch
from hip_attention_b200 import paged_decode_attention, read_status
kc, vc = (torch.randn((64, 16, 2, 64), device='cuda').half() for _ in range(2))
table = torch.zeros((1, {width}), dtype=torch.int32, device='cuda')
table[0, :64] = torch.randperm(64, device='cuda')
q, lens = torch.randn((1, 4, 64), device='cuda').half(), torch.tensor([{n}], device='cuda')
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = paged_decode_attention(q, kc, vc, table, lens)
graph.replay()
assert torch.equal(out, paged_decode_attention(q, kc, vc, table, lens)) and out.abs().sum() > 0 and read_status('cuda') == 0
print('fine')
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("before", ["copy", "fill", "other stream", "kernel", "nothing"])
def test_captured_behind_anything(before):
    """What a captured call reads may come from a copy, a fill, a kernel or another stream."""
    from hip_attention_b200 import paged_decode_attention
    g = torch.Generator(device="cuda").manual_seed(0)
    kc, vc = (torch.randn((64, 16, 2, 64), generator=g, device="cuda") for _ in range(2))
    q, table, lens = torch.randn((1, 4, 64), generator=g, device="cuda"), torch.randperm(64, generator=g, device="cuda")[None], torch.tensor([900], device="cuda")
    want = paged_decode_attention(q, kc, vc, table, lens)
    host, q2, side = q.cpu().pin_memory(), torch.zeros_like(q), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cur = torch.cuda.current_stream()
        if before == "copy":
            q2.copy_(host, non_blocking=True)
        elif before == "other stream":
            side.wait_stream(cur)
            with torch.cuda.stream(side):
                q2.copy_(q)
            cur.wait_stream(side)
        elif before != "nothing":
            torch.mul(q, 1.0, out=q2)
            if before == "fill":
                torch.zeros(4096, device="cuda")
        outs = [paged_decode_attention(q if before == "nothing" else q2, kc, vc, table, lens) for _ in range(2)]
    q2.zero_()
    for _ in range(10):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
