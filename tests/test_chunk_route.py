"""Which calls of kv4_attend_chunk take the kernels for many rows, by the scratch memory that those ask for."""
import pytest

from glint_amd import glint_hip as H


@pytest.mark.parametrize("B,tokens,rows,D,many", [
    (1, 4000, 512, 128, False), (1, 4000, 1024, 128, False), (1, 16000, 256, 128, False), (1, 16000, 1024, 128, True),
    (2, 16000, 192, 128, False), (2, 16000, 512, 128, True), (8, 1000, 256, 128, False), (8, 1000, 512, 128, True),
    (8, 4000, 128, 128, False), (8, 4000, 256, 128, True), (8, 16000, 128, 128, False), (8, 16000, 256, 128, True),
    (32, 1000, 128, 128, False), (32, 1000, 256, 128, True), (32, 4000, 256, 128, True), (1, 16000, 512, 64, False),
    (8, 4000, 512, 64, True)])
def test_rows_and_products(B, tokens, rows, D, many):
    """8 key heads under 32 query heads, as measured: the faster side."""
    size = H.serve_lib().glint_kv4_attend_chunk_scratch(B, rows // 4, 32, 8, D, (tokens + 63) // 64, 0)
    assert size > 0 if many else size == 0


def test_bounds_past_64_bits():
    """The largest bounds that a shape allows: never few rows."""
    assert H.serve_lib().glint_kv4_attend_chunk_scratch((1 << 31) - 1, 1 << 18, 65535, 65535, 128, 1 << 24, 0) != 0
