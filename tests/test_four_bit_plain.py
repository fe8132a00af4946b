"""The 4-bit format itself, on the CPU: what a block rounds to, the page layouts' refusals, and a step's list of pages."""
import numpy as np
import pytest
import torch

import four_bit as F


def test_every_code_is_itself():
    for byte in (8, 100, 127, 252):
        codes = np.concatenate([np.arange(16), np.arange(16)]).astype(np.uint8)
        x = F.numbers(codes[None], np.array([[byte]], dtype=np.uint8))
        c, s, y = F.rounded(x)
        assert s[0, 0] == byte and np.array_equal(y, x) and np.array_equal(c[0], codes)


@pytest.mark.parametrize("top,e", [(4.0, 0), (6.0, 0), (7.0, 0), (7.0001, 1), (7.99, 1), (8.0, 1), (1.0, -2), (0.875, -3), (0.876, -2),
                                   (1e-37, -119), (3.3e38, 125)])
def test_scales(top, e):
    assert F.scale_byte(np.array([0.1 * top, -top])) == e + 127


def test_ties_and_the_largest():
    #  halfway between neighbours: to the even code, that is 0, 1, 1 (not 1.5), 2, 2 (not 3), 4, 4 (not 6); over 6: 6
    x = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.0])
    c, s, y = F.rounded(x[None])
    assert s[0, 0] == 127
    assert y[0].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 0.0, 0.0] and c[0, 8] == 8


def test_off_by_half_a_step_at_most():
    rng = np.random.default_rng(3)
    x = rng.normal(size=(400, 64)) * 10.0 ** rng.uniform(-6, 6, size=(400, 1))
    _, s, y = F.rounded(x)
    unit = np.repeat(2.0 ** (s.astype(float) - 127), 32, axis=1)
    # steps of 2 from 4 on, 1 from 2 on, 0.5 below; what lies from 6 to 7 is cut
    a = np.abs(x) / unit
    step = np.where(a >= 4, 2.0, np.where(a >= 2, 1.0, 0.5))
    assert (np.abs(x - y) <= step / 2 * unit * (1 + 1e-12)).all()
    assert np.array_equal(F.fast_rounded(x)[2], y)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_block_with_no_numbers_reads_as_nan(bad):
    x = np.ones((1, 64))
    x[0, 40] = bad
    _, s, y = F.rounded(x)
    assert s[0].tolist() == [125, 255] and np.isnan(y[0, 32:]).all() and (y[0, :32] == 1).all()


@pytest.mark.parametrize("dim,page,ok", [(64, 64, True), (8, 8, True), (256, 128, True), (80, 32, True), (12, 64, False), (264, 64, False), (64, 48, False), (64, 4, False)])
def test_page_shapes(dim, page, ok):
    from xyntetik_runner_amd.csrc.ops import FourBitPages, KernelError
    if not ok:
        with pytest.raises(KernelError):
            FourBitPages.zeros(3, 2, page, dim, False, "cpu")
        return
    k, v = (FourBitPages.zeros(3, 2, page, dim, values, "cpu") for values in (False, True))
    assert (k.values, v.values, k.page_size, v.page_size, k.heads, k.num_pages) == (False, True, page, page, 2, 3)
    nb = -(-dim // 32)
    assert k.nbytes == v.nbytes == 3 * 2 * page * (dim // 2 + nb)


def test_refused_pages():
    from xyntetik_runner_amd.csrc.ops import FourBitPages, KernelError, Ops
    k, v = (FourBitPages.zeros(3, 2, 64, 64, values, "cpu") for values in (False, True))
    with pytest.raises(KernelError, match="do not fit"):
        FourBitPages(k.codes, k.scales, 96)
    with pytest.raises(KernelError, match="uint8"):
        FourBitPages(k.codes.to(torch.int8), k.scales, 64)
    with pytest.raises(KernelError, match="contiguous"):
        FourBitPages(torch.zeros((3, 2, 64, 64), dtype=torch.uint8)[..., ::2], k.scales, 64)
    assert Ops._pages4("x", k, v, 2, 64, 64)[4] == 3
    for pair, sizes in (((v, k), ()), ((k, k), ()), ((k, torch.zeros(3)), ()), ((k, FourBitPages.zeros(4, 2, 64, 64, True, "cpu")), ()),
                        ((k, v), (4, 64, 64)), ((k, v), (2, 32, 64)), ((k, v), (2, 64, 32))):
        with pytest.raises(KernelError):
            Ops._pages4("x", *pair, *sizes)


@pytest.mark.parametrize("mask,keep", [(None, 0), (40, 0), (40, 33), ("chunk", 0)])
@pytest.mark.parametrize("requests", [None, (2, 0)])
def test_page_list(mask, keep, requests, monkeypatch):
    from xyntetik_runner_amd.cache.manager import RequestCache
    from xyntetik_runner_amd.engine import batch
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda self: self)      # (there is no GPU to pin for)
    real = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, pin_memory=False, **k: real(*a, **k))
    mask = batch.Chunked(64) if mask == "chunk" else mask
    page, starts, lens = 16, [100, 0, 37], [9, 1, 30]
    tables = [[7, 3, 9, 2, 11, 1, 4], [5], [6, 8, 10, 12, 13]]
    held = [RequestCache(b, b, s, [t], False) for b, (s, t) in enumerate(zip(starts, tables))]
    ctx = batch.StepContext(None, "cpu", [batch.StepEntry(b, [0] * n) for b, n in enumerate(lens)], held, 1)
    ctx._held[0][0, 0] = -1 if mask and not keep else ctx._held[0][0, 0]      # (given back)
    slots, table, n = ctx.page_list(0, page, requests, mask, keep)
    slots, table = slots.view(n, 3).tolist(), table.tolist()
    seen = set()
    for b in range(3):
        for i in range(len(table[0])):
            positions = set(range(i * page, min((i + 1) * page, starts[b] + lens[b])))
            wanted = set()
            for p in range(starts[b], starts[b] + lens[b]):
                wanted |= set(range(batch.first_key(mask, p), p + 1)) | (set(range(min(keep, p + 1))) if mask else set())
            if (requests is None or b in requests) and positions & wanted:
                assert slots[table[b][i]] == [b, i, len(positions)]
                seen.add(table[b][i])
            elif not positions or (requests is not None and b not in requests):
                assert table[b][i] == -1
    assert seen == set(range(n))


@pytest.mark.parametrize("mask", [None, 40, "chunk"])
@pytest.mark.parametrize("room", [1, 9, 200])
@pytest.mark.parametrize("G", [1, 4, 24])
def test_row_blocks_cover_every_key_once(mask, room, G):
    """Requests of many rows, 16 of them a block: every block sees its own rows' keys, cut into ranges that meet."""
    from xyntetik_runner_amd.engine.batch import Chunked, few_row_items, first_key
    mask = Chunked(48) if mask == "chunk" else mask
    starts, lens, q0s = [100, 0, 37, 700], [9, 1, 70, 33], [0, 9, 10, 80]
    blocks = [(b, r) for b in range(4) for r in range(0, lens[b] * G, 16)]
    of = [b for b, _ in blocks]
    seen = []

    def ask(tiles):
        seen.append(tiles)
        return room + len(blocks)

    items, _, n_slots = few_row_items(of, [starts[b] for b in of], [lens[b] for b in of], [q0s[b] for b in of], mask, ask, False, first_slot=3,
                                      least=lambda t: 1, row0s=[r for _, r in blocks], group_size=G)
    total, taken = 0, []
    for i, (b, row0) in enumerate(blocks):
        first, last = row0 // G, min(lens[b] - 1, (row0 + 15) // G)
        mine = sorted((it for it in items.tolist() if it[10] == i), key=lambda it: it[2])
        at = first_key(mask, starts[b] + first) // 32 * 32
        total += -(-(starts[b] + last + 1 - at) // 32)
        for it in mine:
            assert it[:2] == [b, row0] and it[2] == at and it[3] > at and it[5:8] == [q0s[b], lens[b], starts[b]] and it[11] == len(mine)
            at = it[3]
        assert at == starts[b] + last + 1
        taken += [it[4] for it in mine if it[4] >= 0]
        assert len(mine) > 1 or mine[0][4] == -1
    assert seen == [total] and sorted(taken) == list(range(3, 3 + n_slots)) and len(items) <= room + len(blocks)


def test_which_requests_are_read_back():
    from xyntetik_runner_amd.engine.batch import FOUR_ROWS, four_row_requests, four_row_slots
    assert four_row_requests([8000] * 64, [1] * 64, 4, None, 8) == list(range(64))
    assert four_row_requests([6144], [2048], 4, None, 8) == [] and four_row_requests([6144, 50], [2048, FOUR_ROWS // 4], 4, None, 8) == [1]
    assert four_row_requests([3488], [512], 4, None, 8) == [0]                  # few blocks for the other kernel
    assert four_row_requests([60000], [512], 4, None, 8) == [] and four_row_requests([60000], [512], 4, 1024, 8) == [0]      # a window leaves little to do
    assert four_row_requests([0], [FOUR_ROWS + 1], 1, None, 32) == [0]
    assert four_row_slots(1500, 8, 256) == 2 * four_row_slots(280, 8, 256) == 512 and four_row_slots(10 ** 6, 8, 512) == 256


def test_pages_keep_their_tensors():
    from xyntetik_runner_amd.csrc.ops import FourBitPages
    pages = FourBitPages.zeros(2, 1, 16, 32, False, "cpu")
    assert pages.pointers == (pages.codes.data_ptr(), pages.scales.data_ptr())
    for name in ("codes", "scales"):
        with pytest.raises(AttributeError):
            setattr(pages, name, torch.zeros(1))
