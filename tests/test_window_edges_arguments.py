"""Refusals of the windowed prefill at the ends of its sizes, without a GPU: before the device is touched."""
import pytest

from vllm_paged_compression_amd import _lib

P = 1 << 20   # stands for an aligned device pointer; nothing dereferences it


def prefill(lib, max_q_len, Hq=4, H=1, D=64, k=P, kv_rows=99):
    return lib.pe_prefill_window(P, P, k, k, P, P, 1, max_q_len, 99, kv_rows, Hq, H, D, Hq * D, H * D, H * D, Hq * D,
                                 0.1, 4, 0, 2, None)


@pytest.mark.parametrize("Hq,H,D,rows", [(4, 1, 64, 64), (4, 4, 32, 64), (3, 1, 64, 64)])
def test_more_row_blocks_than_a_grid_dimension_holds(Hq, H, D, rows):
    """`rows` = the most rows that a workgroup takes; a grid dimension holds 65535 workgroups."""
    lib = _lib.load()
    for n in (65535 * rows + 1, 1 << 22):
        assert prefill(lib, n, Hq, H, D) == 2 and b"grid too large" in lib.pe_last_error(), (n, lib.pe_last_error())


def test_null_rows():
    lib = _lib.load()
    assert prefill(lib, 10, k=None) == 1 and b"null pointer" in lib.pe_last_error()
    assert prefill(lib, 10, k=None, kv_rows=0, D=72) == 2 and b"head size" in lib.pe_last_error()   # past the pointers
