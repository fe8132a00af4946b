"""The limits of a cache in 4 bits, on the CPU: which requests are read back beside the codes."""
import pytest
import torch

from xyntetik_runner_amd.engine import batch


def plain_step(monkeypatch, starts, q_lens, tables):
    from xyntetik_runner_amd.cache.manager import RequestCache
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)      # (there is no GPU to pin for)
    real = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, pin_memory=False, **k: real(*a, **k))
    held = [RequestCache(b, b, s, [t], False) for b, (s, t) in enumerate(zip(starts, tables))]
    return batch.StepContext(None, "cpu", [batch.StepEntry(b, [0] * n) for b, n in enumerate(q_lens)], held, 1)


@pytest.mark.parametrize("most", [0, 5, 9, 10, 14, 15, 40])
def test_requests_that_are_read_back(most):
    rows, pages = [500, 2000, 500, 900, 600], [5, 9, 4, 1, 30]
    got = batch.read_back_requests([0, 1, 2, 3], rows, pages, most)
    assert got == {0: [1], 5: [1], 9: [1], 10: [1, 3], 14: [1, 2, 3], 15: [0, 1, 3], 40: [0, 1, 2, 3]}[most]
    assert batch.read_back_requests([4, 3], rows, pages, most) == ([3, 4] if most == 40 else [3])
    assert batch.read_back_requests([4], rows, pages, most) == [4] and batch.read_back_requests([], rows, pages, most) == []


@pytest.mark.parametrize("mask,keep", [(None, 0), (40, 0), (40, 33), (40, 500), (batch.Chunked(64), 0), (batch.Chunked(64), 20)])
def test_pages_read(mask, keep):
    """As many as hold a key of some row."""
    for start, end, page in ((0, 1, 16), (100, 109, 16), (37, 67, 8), (64, 65, 32), (700, 900, 64), (63, 64, 64)):
        wanted = set()
        for p in range(start, end):
            wanted |= {j // page for j in range(batch.first_key(mask, p), p + 1)} | ({j // page for j in range(min(keep, p + 1))} if mask else set())
        kept, first, last = batch.pages_read(start, end, page, mask, keep)
        assert wanted == set(range(kept)) | set(range(first, last)) and kept <= first


def test_a_step_of_deep_portions_reads_back_no_more_than_the_bound(monkeypatch):
    """Twenty portions of 101 tokens behind 131,072: every one a request of more than 400 rows, 0.54 GB a layer each."""
    heads, group, page, channels = 8, 4, 64, 256
    starts, q_lens = [131072 - 101 * (b + 1) for b in range(20)], [101] * 20
    ctx = plain_step(monkeypatch, starts, q_lens, [list(range(1, 2049))] * 20)
    assert batch.four_row_requests(starts, q_lens, group, None, heads) == []
    page_bytes = heads * page * channels * 2
    plan = ctx.attention_plan(0, group, None, heads, page, few_rows=batch.FEW_FOUR, few_channels=channels, read_back=(2 << 30) // page_bytes)
    assert plan.rest and sum(-(-(starts[b] + 101) // page) for b in plan.rest) * page_bytes <= 2 << 30
    items = plan.few.view(-1, batch.FEW_INTS)
    assert set(items[:, 0].tolist()) == set(range(20)) - set(plan.rest)
    assert ctx.attention_plan(0, group, None, heads, page, few_rows=batch.FEW_FOUR, few_channels=channels).rest == tuple(range(20))


@pytest.mark.parametrize("requests", [(-1,), (0, 3), (2, -3), (1 << 40,)])
def test_requests_that_a_step_does_not_have(requests, monkeypatch):
    """(A place below 0 is one of Python's from the end, and would have been a row before the block table's first on the GPU.)"""
    from xyntetik_runner_amd.csrc.ops import FourBitPages, KernelError, Ops
    ctx = plain_step(monkeypatch, [20, 3, 40], [1, 1, 1], [[1, 2], [3], [4, 5, 6]])
    ops = Ops.__new__(Ops)
    made = []
    monkeypatch.setattr(ctx, "page_list", lambda *a: made.append(a))
    monkeypatch.setattr(Ops, "_here", staticmethod(lambda *a: None))
    pages = [FourBitPages.zeros(8, 1, 16, 32, values, "cpu") for values in (False, True)]
    with pytest.raises(KernelError, match="requests"):
        ops.read_pages(*pages, ctx, 0, torch.bfloat16, requests=requests)
    assert not made
