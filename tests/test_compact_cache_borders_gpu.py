"""Compact caches' operators at the borders of their formats and calls: codes next to a border, rows behind a window, workspaces that hold some rows at a time, results
between padding, tables wider than their rows, values whose groups differ in size."""
from __future__ import annotations

import math

import pytest
import torch

import plain_packed as plain
from test_packed_cache_gpu import DEVICE, HALF, ints, random_pages, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _seed():
    torch.manual_seed(987)


# ---------------------------------------------------------------------------------------
# the write
# ---------------------------------------------------------------------------------------
def sum_of_squares(x):
    """In 32 bits, every addition by itself: 64 channels by halves; others each four channels in order, then halves of those."""
    square = x * x
    if x.shape[-1] != 64:
        a, b, c, d = square.unflatten(-1, (-1, 4)).unbind(-1)
        square = ((a + b) + c) + d
    while square.shape[-1] > 1:
        half = square.shape[-1] // 2
        square = square[..., :half] + square[..., half:]
    return square


def packed_32(x, group):
    """(codes, words) in elementary 32-bit operations."""
    parts = x.unflatten(-1, (-1, group))
    low, high = parts.amin(-1).clamp(max=0.0), parts.amax(-1).clamp(min=0.0)
    bits = (((high - low) / torch.full_like(high, 15.0)).view(torch.int32) + 0x000F_FFFF) & -0x0010_0000
    step = bits.view(torch.float32)
    zero = torch.round(-low / step)
    code = (torch.round(parts / step.unsqueeze(-1)) + zero.unsqueeze(-1)).clamp(0, 15).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), ((bits >> 16) + zero.int()).to(torch.int16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq, nkv, d, group, page", [(32, 8, 128, 64, 256), (4, 8, 128, 32, 64), (6, 8, 64, 32, 24), (2, 4, 256, 128, 16)])
def test_portions_are_packed_bit_for_bit(dtype, nq, nkv, d, group, page):
    """Codes are whole numbers: whoever norms, rotates and packs with the same 32-bit operations finds the same ones, over portions long enough for keys next to a border."""
    from pylon_b200.kernels import ops

    counts, gap = [1024, 1000], 300
    table, pool, _, _, row, slots = tables(counts, counts, page)
    positions = slots + gap
    angles = torch.arange(1024 + gap, device=DEVICE, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d)
    cos, sin = angles.cos().float(), angles.sin().float()
    page_of, at = table.long()[row.long(), slots.long() // page], slots.long() % page
    for _ in range(12):
        q_weight, k_weight = (1 + 0.1 * torch.randn(d, device=DEVICE) for _ in range(2))
        qkv = torch.randn(sum(counts), (nq + 2 * nkv) * d, device=DEVICE).to(dtype)
        k_pages, v_pages = (ops.packed_pages(pool, nkv, page, d, group, DEVICE) for _ in range(2))
        q = ops.qk_norm_rope_slot_write(qkv, q_weight, k_weight, 1e-6, cos, sin, d, positions, row, table, page, k_pages, v_pages, nq, nkv, d, slots=slots)
        x = qkv.float().view(-1, nq + 2 * nkv, d)
        qk = x[:, : nq + nkv]
        qk = qk * torch.rsqrt(sum_of_squares(qk) * (1.0 / d) + 1e-6) * torch.cat((q_weight.expand(nq, d), k_weight.expand(nkv, d)))
        c, s = cos[positions.long()][:, None], sin[positions.long()][:, None]
        first, second = qk[..., : d // 2], qk[..., d // 2 :]
        qk = torch.cat((first * c - second * s, second * c + first * s), dim=-1)
        assert torch.equal(q, qk[:, :nq].flatten(1).to(dtype))
        for pages, values in ((k_pages, qk[:, nq:]), (v_pages, x[:, nq + nkv :])):
            codes, words = packed_32(values, group)
            assert torch.equal(pages.words[page_of, :, at], words) and torch.equal(pages.codes[page_of, :, at], codes)
    ops.raise_on_kernel_errors(torch.device(DEVICE))
