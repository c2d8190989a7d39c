"""The paged attention of pieces without a GPU: how much one call takes."""
import pytest

from sile_amd import _abi
from tests.test_serving_abi import CHUNK, refused
from tests.test_serving_overlaps import passes

FAR = 1 << 40
LARGE = {**CHUNK, "n_rows": 1, "n_tokens": 2 ** 30 - 1, "q_heads": 2, "kv_heads": 2, "head_dim": 8, "q": FAR, "ldq": 16, "o": 2 * FAR, "ldo": 16,
         "num_pages": 8, "page_stride": 256}


def test_units():
    """2^24 units would be a launch of 2^32 threads; 16 fewer (of two key heads) are one call."""
    refused("Shape", _abi.paged_attn_chunk, **LARGE)
    assert "too many for one call" in _abi.last_error()
    passes(_abi.paged_attn_chunk, **{**LARGE, "n_tokens": 2 ** 30 - 8 * 128})


@pytest.mark.parametrize("change", [dict(ldq=1 << 41), dict(ldo=1 << 41), dict(ldq=1 << 62), dict(n_tokens=2 ** 30 - 8 * 128, ldo=1 << 16)])
def test_leading_dimensions(change):
    """Offsets of a call's tokens stay below 2^46 elements."""
    refused("Shape", _abi.paged_attn_chunk, **{**LARGE, "n_tokens": 30, **change})
    assert "leading dimension" in _abi.last_error()
