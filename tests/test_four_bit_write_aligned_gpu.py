"""Writing 4-bit pages from rows of 16-byte pieces, whose kernel reads and rotates eight channels at a time, against plain numpy in 64 bits."""
import numpy as np
import pytest
import torch

import four_bit as F
from test_four_bit_gpu import DEV, DT, WRITES, host, on_gpu, ops, rotated, scattered, step          # noqa: F401 (ops: the fixture)

pytestmark = pytest.mark.gpu

ALIGNED = WRITES + [
    # H, Hk, D, Dv, rot, interleaved, paired, page, starts, q_lens
    (3, 2, 96, 96, 96, True, False, 32, [13, 0], [30, 9]),                    # pairs side by side, of whole heads
    (2, 2, 128, 64, 40, True, False, 64, [4000], [19]),                       # and of a part of a head
    (4, 1, 80, 80, 48, False, False, 16, [9], [20]),                          # halves of a part of a head, a last block of 16
    (3, 3, 112, 112, 112, False, True, 16, [0, 65530], [11, 9]),              # in paired order, a last block of 16
    (2, 1, 256, 256, 128, False, True, 128, [120], [24]),
]


@pytest.mark.parametrize("more", [0, 4])
@pytest.mark.parametrize("case", ALIGNED)
@pytest.mark.parametrize("dt", ["bfloat16", "float32"])
def test_write_of_aligned_rows(ops, case, dt, more):
    from xyntetik_runner_amd.csrc.ops import paired_order
    H, Hk, D, Dv, rot, interleaved, paired, page, starts, q_lens = case
    rng = np.random.default_rng(D + rot + len(starts) + 1)
    tables, n_pages = scattered(rng, [s + n for s, n in zip(starts, q_lens)], page)
    ctx = step(starts, q_lens, tables)
    T, QK = sum(q_lens), (H + Hk) * D
    inv = (1.0 / 10000.0 ** (np.arange(0, rot, 2) / max(rot, 1))).astype(np.float32)
    x = (rng.normal(size=(T, QK + Hk * Dv + more)) * np.exp(rng.normal(size=(T, 1)))).astype(np.float32)
    nothing = [[np.zeros((0, Hk, d), dtype=np.uint8)] * 3 for d in (D, Dv)]
    kp, vp = (on_gpu(*F.fill_pages([e] * len(q_lens), tables, n_pages, page, values, junk=rng), d) for e, values, d in zip(nothing, (False, True), (D, Dv)))
    proj = torch.tensor(x, device=DEV)
    assert proj.stride(0) % 4 == 0 and QK % 4 == 0
    q = torch.full((T, H * D), 7.0, dtype=DT[dt], device=DEV)
    ops.rope_kv_write(proj[:, :H * D] if H else None, proj[:, H * D:QK], proj[:, QK:QK + Hk * Dv], q if H else None, kp, vp, ctx.positions, ctx.req_of_token,
                      ctx.block_table(0), torch.tensor(inv, device=DEV) if rot else None, H, Hk, D, rot, interleaved, 0.75, page, paired=paired)
    x64 = x.astype(np.float64)
    qk = x64[:, :QK].reshape(T, H + Hk, D)
    if paired:
        plain = np.empty_like(qk)
        plain[..., paired_order(D, rot)] = qk
        qk = plain
    want, size = rotated(qk, ctx.positions.cpu().numpy(), inv, rot, interleaved, 0.75)
    # half a step of the type, and of 32 bits: cosine, sine (2 steps each from the angle on), two products and a sum
    slack = 8 * 2.0 ** -24 * size
    if H:
        eps = 2.0 ** -8 if dt == "bfloat16" else 0.0
        assert (np.abs(q.cpu().double().numpy().reshape(T, H, D) - want[:, :H]) <= eps * np.abs(want[:, :H]) + slack[:, :H]).all()
    v64 = x64[:, QK:QK + Hk * Dv].reshape(T, Hk, Dv)
    row = 0
    for b, n in enumerate(q_lens):
        places = list(range(starts[b], starts[b] + n))
        got = F.pages_rows(*host(vp), tables[b], places, page, True)
        assert np.array_equal(got, F.rounded(v64[row:row + n])[2])              # (no rotation: exactly the oracle's)
        codes, scales = host(kp)
        got, ref, off = F.pages_rows(codes, scales, tables[b], places, page, False), want[row:row + n, H:], slack[row:row + n, H:]
        at = np.array([[tables[b][p // page], p % page] for p in places])
        byte = scales[at[:, 0], :, at[:, 1] // 8, :, at[:, 1] % 8].astype(np.float64)
        unit = np.repeat(2.0 ** (byte - 127), 32, axis=-1)[..., :D]
        a = np.abs(ref) / unit
        # half a step of the numbers, and as much more as the rotated one itself is off by 32-bit arithmetic
        assert (np.abs(got - ref) <= np.where(a >= 4, 2.0, np.where(a >= 2, 1.0, 0.5)) * unit / 2 + off + 1e-12 * np.abs(ref)).all()
        for block in range(scales.shape[3]):
            part = slice(32 * block, 32 * block + 32)
            least, most = (np.array([[F.scale_byte(r[part]) for r in tok] for tok in t]) for t in (np.maximum(np.abs(ref) - off, 0), np.abs(ref) + off))
            assert ((least <= byte[..., block]) & (byte[..., block] <= most)).all()
        row += n


@pytest.mark.parametrize("more", [0, 1])          # (an odd stride: the kernel that reads channel by channel)
@pytest.mark.parametrize("start", [0, 60000, 130000])
def test_cosines_and_sines_next_to_their_zeros(ops, start, more):
    """Queries (1, 0) turn into the angle's cosine and sine.  Of each number: four steps for the function, as OpenCL's table of errors allows it, half a step each
    for what is put back, the scale and the product, 6 * 2^-23 in all; and the angle itself, up to 21,000 turns that are rounded in 64 bits twice, 2^-52 of them each."""
    from xyntetik_runner_amd.csrc.ops import FourBitPages
    n, D, page = 700, 128, 64
    ctx = step([start], [n], [[0] * (start // page) + list(range(1, 13))])
    inv = (1.0 / 10000.0 ** (np.arange(0, D, 2) / D)).astype(np.float32)
    x = torch.zeros((n, 3 * D + more), device=DEV)
    x[:, :D // 2] = 1.0
    q = torch.empty((n, D), device=DEV)
    kp, vp = (FourBitPages.zeros(13, 1, page, D, values, DEV) for values in (False, True))
    ops.rope_kv_write(x[:, :D], x[:, D:2 * D], x[:, 2 * D:3 * D], q, kp, vp, ctx.positions, ctx.req_of_token, ctx.block_table(0), torch.tensor(inv, device=DEV),
                      1, 1, D, D, False, 1.0, page)
    angle = np.arange(start, start + n)[:, None] * inv.astype(np.float64)
    want = np.concatenate([np.cos(angle), np.sin(angle)], axis=1)
    assert np.abs(want)[:, :-1].min() < 1e-4                # (some lie next to a zero)
    assert (np.abs(q.cpu().double().numpy() - want) <= 6 * 2.0 ** -23 * np.abs(want) + 2 * np.abs(np.tile(angle, 2)) * 2.0 ** -52 + 2.0 ** -50).all()
