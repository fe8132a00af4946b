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


def ref_without(q, k, v, start, missing, Hk, scale, window, sinks):
    """Rows of one request over the keys that exist."""
    n, H, D = q.shape
    out = np.zeros((n, H, v.shape[2]))
    for i in range(n):
        p = start + i
        js = [j for j in range(max(0, p - window + 1) if window else 0, p + 1) if j not in missing]
        for h in range(H):
            s = k[js, h // (H // Hk)] @ q[i, h] * scale
            top = max(s.max(initial=-np.inf), sinks[h] if sinks is not None else -np.inf)
            if top == -np.inf:
                continue
            e = np.exp(s - top)
            out[i, h] = e @ v[js, h // (H // Hk)] / (e.sum() + (np.exp(sinks[h] - top) if sinks is not None else 0.0))
    return out


@pytest.mark.parametrize("bad", [-1, 0, 1 << 30, "past the table"])
@pytest.mark.parametrize("dt", ["bfloat16", "float32"])
@pytest.mark.parametrize("path", ["codes", "read back", "recorded"])
@pytest.mark.parametrize("H,Hk,D,window,q_lens", [(8, 2, 64, None, [1, 1, 1]), (4, 1, 128, None, [9, 5, 3]), (4, 2, 72, 90, [1, 2, 1]), (16, 2, 64, 150, [100, 130, 3]),
                                                  (4, 2, 80, None, [40, 6, 2])])
def test_pages_that_do_not_exist_are_left_out(ops, bad, dt, path, H, Hk, D, window, q_lens, monkeypatch):
    """A page that a row's keys would lie in and that the cache does not have, some of a request's or all: its keys are in no row's sum, whichever kernel runs
    and whatever page 0 holds (here blocks that read as NaN)."""
    from xyntetik_runner_amd.engine import batch
    monkeypatch.setattr(batch, "four_row_requests", lambda starts, *a: [] if path == "read back" else list(range(len(starts))))
    rng, page, starts = np.random.default_rng(D + H), 32, [200, 150, 60]
    lens = [s + n for s, n in zip(starts, q_lens)]
    counts = [-(-n // page) for n in lens]
    ids = (rng.permutation(sum(counts)) + 1).tolist()
    full = [[ids.pop() for _ in range(c)] for c in counts]
    n_pages = sum(counts) + 1
    ks, vs = ([F.random_sequence(rng, n, Hk, D) for n in lens] for _ in range(2))
    pages = []
    for seqs, values in ((ks, False), (vs, True)):
        codes, scales = F.fill_pages(seqs, full, n_pages, page, values, junk=rng)
        scales[0] = 255
        pages.append(on_gpu(codes, scales, D))
    gone = [{2} if bad != "past the table" else {counts[0] - 1}, set(), set(range(counts[2]))]      # (the first request's table is the longest)
    none = {0: n_pages, "past the table": -1}.get(bad, bad)
    tables = [[none if i in g else p for i, p in enumerate(t)] for t, g in zip(full, gone)]
    if bad == "past the table":
        tables[0].pop()
    ctx = step(starts, q_lens, tables)
    scale, sinks = D ** -0.5, (rng.normal(size=H).astype(np.float32) if window else None)
    q = [torch.tensor(rng.normal(size=(n, H, D)) * 1.5).to(DT[dt]) for n in q_lens]
    got = ops.attention(torch.cat(q).reshape(-1, H * D).contiguous().to(DEV), *pages, Recorded(ctx) if path == "recorded" else ctx, 0, H, Hk, D, page, scale, window,
                        sinks=torch.tensor(sinks, device=DEV) if window else None).cpu().double().numpy().reshape(-1, H, D)
    want = np.concatenate([ref_without(q[b].double().numpy(), ks[b][2], vs[b][2], starts[b], {j for i in gone[b] for j in range(page * i, page * i + page)}, Hk, scale, window, sinks)
                           for b in range(3)])
    assert np.isfinite(got).all() and not got[q_lens[0] + q_lens[1]:].any()
    # (bounds as in the tests of attention over pages that exist: two roundings to bfloat16, or sums in 32 bits)
    assert np.abs(got - want).max() <= (1.2e-2 if dt == "bfloat16" else 2e-5) * np.abs(want).max()


@pytest.mark.parametrize("columns", ["fewer than the rows are apart", "shared by all requests"])
def test_block_tables_that_are_views(ops, columns):
    """A table of some columns of a wider one, or of one row that all requests read: a position past its columns has no page."""
    from xyntetik_runner_amd.csrc.ops import FourBitPages
    rng, page, Hk, D, B = np.random.default_rng(4), 16, 2, 32, 3
    wide = torch.arange(1, 13, dtype=torch.int32, device=DEV).view(B, 4)
    table = wide[:, :2] if columns.startswith("fewer") else wide[:1, :2].expand(B, 2)
    assert not table.is_contiguous()
    pos = [0, 15, 16, 31, 32, 33, 47, 48, 5, 21, 40, 63, 64, 2, 30, 35, 3, 36, 37, 38]
    req = [0] * 8 + [1] * 5 + [2] * 7
    p, r = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (pos, req))
    x = torch.tensor(rng.normal(size=(len(pos), 2 * D)), dtype=torch.float32, device=DEV)
    h = torch.tensor(rng.normal(size=(len(pos), 64)), device=DEV).bfloat16()
    w = torch.tensor(rng.normal(size=(6 * D, 64)), device=DEV).bfloat16()
    rows = []
    for t in (table, table.contiguous()):
        for fused in (False, True):
            kp, vp = (FourBitPages.zeros(14, Hk, page, D, values, DEV) for values in (False, True))
            if fused:                    # 20 rows: the kernel that adds the product's ranges up writes
                ops.project_rope_kv_write(h, w, None, kp, vp, p, r, t, None, 2, Hk, D, 0, False, 1.0, page)
            else:
                ops.rope_kv_write(None, x, x, None, kp, vp, p, r, t, None, 0, Hk, D, 0, False, 1.0, page)
            mine = torch.unique(table).tolist()
            assert all(not pages.scales[i].any() for pages in (kp, vp) for i in range(14) if i not in mine)
            k, v = ops.read_rows(kp, vp, p, r, t, torch.float32)
            for got in (k, v):
                there = torch.tensor([q < 2 * page for q in pos], device=DEV)
                assert got[there].abs().amax(1).min() > 0 and not got[~there].any()
            kp.scales.fill_(127)
            kp.codes.fill_(0x22)
            rows += [k, v, *ops.read_rows(kp, vp, p, r, t, torch.float32)]
    for a, b in zip(rows[:8], rows[8:]):
        assert torch.equal(a, b)
