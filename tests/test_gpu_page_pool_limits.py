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
