"""The limits of a cache in 4 bits: how much is read back at once, pages that do not exist, block tables that are views, requests that a step does not have."""
import numpy as np
import pytest
import torch

import four_bit as F
from test_four_bit_gpu import DEV, DT, Recorded, attend, on_gpu, ops, scattered, step          # noqa: F401 (ops: the fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture
def read(ops, monkeypatch):
    """Bytes of every set of pages that is read back."""
    got, real = [], ops.read_pages

    def noted(*a, **k):
        pages = real(*a, **k)
        got.append(pages[0].nbytes + pages[1].nbytes)
        return pages

    monkeypatch.setattr(ops, "read_pages", noted)
    return got


@pytest.mark.parametrize("what", [{}, dict(sinks=True, slopes=True), dict(cap=1.3)])
@pytest.mark.parametrize("mask", [None, 100])
@pytest.mark.parametrize("pages,most", [(0, 10), (16, 16), (26, 26), (27, 27), (1000, 27)])
def test_what_is_read_back_beside_the_codes(ops, read, mask, pages, most, what, monkeypatch):
    """Requests that would all be read back: up to the bound, or one of more; the others from the codes, with the same results."""
    from xyntetik_runner_amd.engine import batch
    monkeypatch.setattr(batch, "four_row_requests", lambda *a: [])
    H, Hk, D, page = 16, 2, 64, 32
    page_bytes = Hk * page * 2 * D * 2
    monkeypatch.setattr(ops, "READ_BACK_BYTES", pages * page_bytes + 5)
    attend(ops, (H, Hk, D, D, page, mask, [300, 37, 100], [60, 260, 30]), "bfloat16", 600 + pages, **what)      # 12, 10 and 5 pages without a mask
    assert read and max(read) <= most * page_bytes
    if not mask:
        assert max(read) == {0: 10, 16: 15, 26: 22, 27: 27, 1000: 27}[pages] * page_bytes


@pytest.mark.parametrize("mask", [50, "chunk"])
@pytest.mark.parametrize("pages", [40, 1000])
def test_kept_pages_count_among_what_is_read_back(ops, read, mask, pages, monkeypatch):
    """A window leaves few pages to read, the first keys that are kept beside it many."""
    from xyntetik_runner_amd.engine.batch import Chunked
    H, Hk, D, page = 4, 2, 80, 16
    page_bytes = Hk * page * 2 * D * 2
    monkeypatch.setattr(ops, "READ_BACK_BYTES", pages * page_bytes)
    attend(ops, (H, Hk, D, D, page, Chunked(64) if mask == "chunk" else mask, [900, 700], [40, 1]), "bfloat16", 700, keep=500)
    assert all(n <= pages * page_bytes for n in read) and bool(read) == (pages == 1000)


def test_one_request_of_more_is_read_back(ops, read, monkeypatch):
    monkeypatch.setattr(ops, "READ_BACK_BYTES", 1000)
    attend(ops, (4, 2, 80, 80, 16, None, [100], [40]), "bfloat16", 710)
    assert read and set(read) == {9 * 2 * 16 * 2 * 80 * 2}
