"""GPU: the attention of pieces of prompts with pages of every size, and none, over keys that are shared
out to workgroups."""
import pytest

from tests.test_gpu_paged_chunk import Case, run_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8,d,page", [(False, 128, 16), (True, 64, 16), (False, 64, 1)])
def test_rows_without_pages(hip, fp8, d, page):
    """Long rows of which no page is there: zeros, beside rows as they are."""
    case = Case(d, "bf16", [(8, 6000), (5, 700), (40, 5000), (1, 6000)], 4, 1, d, page, fp8=fp8)
    gone = {i: set(range(6000 // page + 1)) for i in (0, 2, 3)}
    for i in gone:
        case.tables[i] = -1
    run_case(hip, case, f"chunk rows without pages fp8={fp8} d {d} pages of {page}", gone=gone)
    got = case.result(hip)
    for i in gone:
        assert (got[case.starts[i]:case.starts[i + 1]] == 0).all()
