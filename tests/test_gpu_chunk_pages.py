"""GPU: the attention of pieces of prompts with pages of every size, and none, over keys that are shared
out to workgroups."""
import numpy as np
import pytest

from tests.test_gpu_paged_chunk import NAN16, Case, as_f32, run_case, say

pytestmark = pytest.mark.gpu

# pages smaller than the keys of one load (512 elements) and the least that are not, of 16-bit caches; 8-bit ones
PAGES = [("f16", False, 64, 1), ("bf16", False, 64, 4), ("f16", False, 64, 8), ("bf16", False, 128, 1), ("f16", False, 128, 2),
         ("bf16", False, 128, 4), ("f16", False, 256, 1), ("bf16", False, 256, 2), ("f16", True, 64, 1), ("bf16", True, 64, 128),
         ("bf16", True, 128, 1), ("f16", True, 128, 8), ("bf16", True, 256, 8), ("f16", True, 256, 128)]


@pytest.mark.parametrize("dtype,fp8,d,page", PAGES)
def test_over_workgroups(hip, dtype, fp8, d, page):
    """Long rows beside short ones, tiles of several pieces and of a few tokens in one share."""
    case = Case(d + page, dtype, [(3, 3000), (1, 20), (60, 1500), (1, 2001), (0, 700), (2, 1)], 4, 2, d, page, fp8=fp8)
    run_case(hip, case, f"chunk over workgroups {dtype} fp8={fp8} d {d} pages of {page}")


@pytest.mark.parametrize("dtype,fp8,d,page", PAGES)
def test_window_over_workgroups(hip, dtype, fp8, d, page):
    case = Case(d + page + 1, dtype, [(40, 2500), (1, 3000), (7, 1900)], 4, 1, d, page, fp8=fp8, window=700, sinks=5)
    run_case(hip, case, f"chunk windows over workgroups {dtype} fp8={fp8} d {d} pages of {page}", heads=[0, 3])


@pytest.mark.parametrize("dtype,fp8,d,page", PAGES)
def test_drafts(hip, dtype, fp8, d, page):
    """A few tokens behind many, missing pages, and a NaN that only a row's last token sees."""
    case = Case(d + page + 2, dtype, [(6, 1501), (1, 900), (8, 4000), (4, 4)], 4, 1, d, page, fp8=fp8)
    gone = {0: {90 * 16 // page, 93 * 16 // page}, 2: {0, 2000 // page, 3900 // page}}
    gone = {i: {e for e in entries if e != (case.seqs[i][1] - 1) // page} for i, entries in gone.items()}
    for i, entries in gone.items():
        for e in entries:
            case.tables[i, e] = (-1, case.num)[e % 2]
    for i in (0, 2, 3):
        n = case.seqs[i][1] - 1
        for pool in case.pools:
            view = pool[:, :case.hkv * page * d].reshape(case.num, case.hkv, page, d)
            view[case.tables[i, n // page], :, n % page] = 0x7F if fp8 else NAN16[dtype]
    say(f"chunk drafts {dtype} fp8={fp8} d {d} pages of {page}")
    case.upload(hip)
    case.run(hip)
    got = as_f32(case.result(hip), dtype)
    for i in (0, 2, 3):
        assert np.isnan(got[case.starts[i + 1] - 1]).all(), "the token of the NaN key"
    case.seqs = [(new - (i != 1), n - (i != 1)) for i, (new, n) in enumerate(case.seqs)]
    case.check(case.do.download(np.uint16, (case.n + 1, case.ldo))[:case.n, :case.hq * d].reshape(case.n, case.hq, d),
               "drafts", gone=gone)


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
