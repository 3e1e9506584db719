"""slm_paged.h without a GPU: calls without a context or cache are refused, and
NULL handles are harmless."""
import ctypes

from slm_testlib import load_product

P = load_product()


def test_null_handles():
    lib = P.load_library()
    out = ctypes.c_void_p(1)
    cfg = P.PagedConfigC(1, 4, 16, 0, 4)
    assert lib.slm_paged_create(None, ctypes.byref(cfg), ctypes.byref(out)) == P.ERR_ARG
    assert not out.value
    assert b"ctx is NULL" in lib.slm_attn_last_error(None)
    assert lib.slm_paged_create(None, ctypes.byref(cfg), None) == P.ERR_ARG
    batch = P.PagedBatch(1, 16, 1, 16, 16)
    assert lib.slm_paged_append_dev(None, None, 0, batch.ref, 16, 16, 16, None, None, 1e-5,
                                    32) == P.ERR_ARG
    assert lib.slm_paged_attend_dev(None, None, 0, batch.ref, 16, 0, 0, 32) == P.ERR_ARG
    lib.slm_paged_destroy(None)
    assert lib.slm_paged_device_ptr(None) is None
    assert lib.slm_paged_offset(None, 0, 0, 0, 0, 0) == ctypes.c_size_t(-1).value


def test_a_batch_is_the_headers_struct():
    # five int32, padded, and three pointers; n_rows and row_start default to one row per sequence
    b = P.PagedBatch(3, 0x1000, 7, 0x2000, 90)
    assert ctypes.sizeof(P.PagedBatchC) == 4 * 4 + 3 * 8 and ctypes.sizeof(P.PagedConfigC) == 20
    assert (b.c.n_seqs, b.c.n_rows, b.c.max_len, b.c.table_stride) == (3, 3, 90, 7)
    assert (b.c.page_table, b.c.lens, b.c.row_start) == (0x1000, 0x2000, None)
