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


# ---------------------------------------------------------------------------------------
# attention over unpacked contexts
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("nq, nkv, d, counts, lengths", [
    (4, 2, 96, [64, 1, 9, 40], [700, 650, 9, 300]), (2, 2, 256, [1, 30, 30, 30], [600, 30, 500, 77]), (8, 1, 32, [20], [900]), (4, 2, 64, [64, 1, 9, 40], [700, 650, 9, 300]),
])
def test_rows_that_are_unpacked_a_few_at_a_time(nq, nkv, d, counts, lengths, known, monkeypatch):
    """Every batch of rows leaves the others' results, and padding tokens' rows, as they are, also where few query tiles over long contexts are cut into parts."""
    from pylon_b200.kernels import ops

    page, bound, tokens = 16, 2000, sum(counts)
    table, pool, q_start, kv_len, row, slots = tables(counts, lengths, page)
    k_pages, v_pages = random_pages(pool, nkv, page, d, 32), random_pages(pool, nkv, page, d, 32)
    q = torch.randn(tokens + 3, nq * d, device=DEVICE).bfloat16()
    row, slots = torch.cat((row, ints([-1] * 3))), torch.cat((slots, ints([0] * 3)))
    expected, size = plain.attention(q[:tokens], k_pages, v_pages, counts, lengths, table, nq, d ** -0.5)
    for rows_at_once in (len(counts), 3, 1):
        monkeypatch.setattr(ops, "UNPACKED_BYTES", rows_at_once * 32 * 64 * nkv * d * 4)
        out = torch.full((tokens + 3, nq * d), 3.0, device=DEVICE).bfloat16()
        for before in (None, float("nan")):      # what fresh memory held before reaches nobody
            torch.full((1 << 24,), 0.0 if before is None else before, device=DEVICE)
            ops.paged_attention_packed(q, k_pages, v_pages, slots, row, q_start, kv_len, table, nq, max(counts), bound, out=out, row_tokens=tuple(counts) if known else None)
            assert (out[tokens:] == 3.0).all()
            # weights of 8 bits and the result's rounding; scores in 32 bits
            assert ((out[:tokens].double() - expected).abs() <= HALF[torch.bfloat16] * (expected.abs() + size) + 2.0 ** -14 * size).all()
    ops.raise_on_kernel_errors(torch.device(DEVICE))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq, nkv, d, page, counts, lengths, window", [
    (8, 2, 128, 16, [1, 2, 1], [700, 301, 40], 100), (8, 2, 128, 24, [1, 1], [700, 301], 33), (8, 2, 64, 256, [1, 1], [900, 1025], 1), (8, 2, 128, 64, [40, 1], [800, 500], 90),
    (4, 2, 64, 7, [70], [500], 128), (8, 2, 96, 16, [1, 30], [700, 900], 65), (32, 8, 128, 64, [200], [4600], 300),
])
def test_pages_that_a_window_has_passed_are_gone(dtype, nq, nkv, d, page, counts, lengths, window):
    """A cache gives back the pages that no token sees any more; the table holds -1 in their places, which is no error and no page."""
    from pylon_b200.kernels import ops

    table, pool, q_start, kv_len, row, slots = tables(counts, lengths, page)
    k_pages, v_pages = random_pages(pool, nkv, page, d, 32), random_pages(pool, nkv, page, d, 32)
    q = torch.randn(sum(counts), nq * d, device=DEVICE).to(dtype)
    gone = table.clone()
    for r, (count, length) in enumerate(zip(counts, lengths)):
        first = max(0, length - count - window + 1) // page
        assert first > 0 or length < window + count
        gone[r, :first] = -1
    expected, size = plain.attention(q, k_pages, v_pages, counts, lengths, table, nq, d ** -0.5, window)
    for row_tokens in (None, tuple(counts)):
        results = [ops.paged_attention_packed(q, k_pages, v_pages, slots, row, q_start, kv_len, each, nq, max(counts), max(lengths), window=window, row_tokens=row_tokens)
                   for each in (table, gone)]
        ops.raise_on_kernel_errors(torch.device(DEVICE))
        assert torch.equal(*results)
        assert ((results[1].double() - expected).abs() <= HALF[dtype] * (expected.abs() + size) + 2.0 ** -14 * size).all()
    # a page that a token sees is still missed
    last = max(0, lengths[0] - counts[0] - window + 1) // page
    gone[0, last] = -1
    ops.paged_attention_packed(q, k_pages, v_pages, slots, row, q_start, kv_len, gone, nq, max(counts), max(lengths), window=window, row_tokens=tuple(counts))
    with pytest.raises(ops.KernelError, match="attention"):
        ops.raise_on_kernel_errors(torch.device(DEVICE))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts, lengths, d", [([1, 2], [300, 40], 64), ([40, 1], [90, 700], 128), ([40, 1], [90, 700], 96)])
def test_padding_rows_of_a_result_anywhere_in_memory(counts, lengths, d, dtype):
    """A result that does not start on 16 bytes is worked out elsewhere: padding tokens' rows are left alone all the same."""
    from pylon_b200.kernels import ops

    nq, nkv, page, tokens = 8, 2, 16, sum(counts)
    table, pool, q_start, kv_len, row, slots = tables(counts, lengths, page)
    k_pages, v_pages = random_pages(pool, nkv, page, d, 32), random_pages(pool, nkv, page, d, 32)
    q = torch.randn(tokens + 2, nq * d, device=DEVICE).to(dtype)
    row, slots = torch.cat((row, ints([-1, -1]))), torch.cat((slots, ints([0, 0])))
    torch.full((1 << 24,), float("nan"), device=DEVICE)      # what fresh memory holds
    out = torch.full(((tokens + 2) * nq * d + 1,), 3.0, dtype=dtype, device=DEVICE)[1:].view(tokens + 2, nq * d)
    assert ops.paged_attention_packed(q, k_pages, v_pages, slots, row, q_start, kv_len, table, nq, max(counts), max(lengths), out=out).data_ptr() == out.data_ptr()
    wanted = ops.paged_attention_packed(q, k_pages, v_pages, slots, row, q_start, kv_len, table, nq, max(counts), max(lengths))
    assert (out[tokens:] == 3.0).all() and torch.equal(out[:tokens], wanted[:tokens])
    ops.raise_on_kernel_errors(torch.device(DEVICE))


@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 96), (torch.bfloat16, 128), (torch.float32, 64)])
def test_rows_that_the_host_knows_to_be_empty(dtype, d):
    """A padded step whose rows all are without tokens."""
    from pylon_b200.kernels import ops

    k_pages, v_pages = random_pages(3, 2, 16, d, 32), random_pages(3, 2, 16, d, 32)
    out, nothing = torch.full((2, 4 * d), 3.0, dtype=dtype, device=DEVICE), ints([-1, -1])
    for max_q in (1, 40):
        for held in (0, 20):
            ops.paged_attention_packed(torch.zeros_like(out), k_pages, v_pages, ints([0, 0]), nothing, ints([0, 0, 0]), ints([held, held]), ints([[0, 1], [2, 0]]), 4, max_q, 32, out=out, row_tokens=(0, 0))
    assert (out == 3.0).all()
    ops.raise_on_kernel_errors(torch.device(DEVICE))


# ---------------------------------------------------------------------------------------
# eviction
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("length, width", [(300, 1_500_000 // 16), (4096, 500_000 // 16), (4000, 1_500_000 // 16), (30_000, 1_500_000 // 16)])
def test_short_rows_of_wide_tables(length, width):
    """Tables of up to 1.5 million slots to a row are taken, however short the rows are."""
    from pylon_b200.kernels import ops

    nkv, page, keep = 2, 16, 100
    table, pool, _, kv_len, _, _ = tables([0], [length], page)
    mass = torch.rand(pool, nkv, page, device=DEVICE)
    places = torch.zeros(pool, nkv, page, dtype=torch.int32, device=DEVICE)
    where, at = plain.row_slots(table[0], length, page)
    for head in range(nkv):
        places[where, head, at] = torch.randperm(length, device=DEVICE).int()
    rows = torch.randn(pool, nkv, page, 3, device=DEVICE)
    expected = plain.evict(mass, places, (rows,), [length], table, keep, 4, 8)
    wide = torch.full((1, width), -1, dtype=torch.int32, device=DEVICE)
    wide[:, : table.shape[1]] = table
    held = ops.evict_slots(mass, places, (rows,), kv_len, wide, length, keep, keep_first=4, keep_recent=8)
    assert held.tolist() == [keep] and all(torch.equal(got, wanted) for got, wanted in zip((mass, places, rows), expected))
    ops.raise_on_kernel_errors(torch.device(DEVICE))


# ---------------------------------------------------------------------------------------
# workspaces
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq, nkv, d, counts, longest, known", [
    (32, 8, 128, [1] * 16, 40_000, True), (32, 8, 128, [1] * 3 + [500], 40_000, True), (32, 8, 128, [1] * 3 + [500], 40_000, False), (8, 2, 96, [1] * 5 + [100, 20], 9_000, True),
    (16, 2, 64, [1] * 40 + [30], 70_000, False), (8, 8, 256, [4, 4], 2_000, True), (4, 2, 64, [1], 300_000, True),
])
def test_what_is_taken_for_a_while(dtype, nq, nkv, d, counts, longest, known):
    """An engine leaves this much free for the operators of a compact cache: calls that are planned for the longest contexts take no more."""
    from pylon_b200.kernels import ops

    page, rows, tokens, votes = 256, len(counts), sum(counts), 64
    lengths = [count + 20 for count in counts]
    table, pool, q_start, kv_len, row, slots = tables(counts, lengths, page)
    wide = torch.zeros(rows, -(-longest // page), dtype=torch.int32, device=DEVICE)
    wide[:, : table.shape[1]] = table
    k_pages, v_pages = random_pages(pool, nkv, page, d, 32), random_pages(pool, nkv, page, d, 32)
    q, out = torch.randn(tokens, nq * d, device=DEVICE).to(dtype), torch.zeros(tokens, nq * d, dtype=dtype, device=DEVICE)
    mass = torch.zeros(pool, nkv, page, device=DEVICE)
    sms = ops._multiprocessors(torch.device(DEVICE))

    def peak(call):
        call()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        call()
        return torch.cuda.max_memory_allocated() - before

    attention = peak(lambda: ops.paged_attention_packed(q, k_pages, v_pages, slots, row, q_start, kv_len, wide, nq, max(counts), longest, out=out, row_tokens=tuple(counts) if known else None))
    masses = peak(lambda: ops.attention_mass(q, k_pages, mass, q_start, kv_len, wide, nq, max(counts), longest, last=votes))
    plain_masses = peak(lambda: ops.attention_mass(q, torch.zeros_like(k_pages.codes).new_zeros((pool, nkv, page, d)).to(dtype), mass, q_start, kv_len, wide, nq, max(counts), longest, last=votes))
    plain_masses -= pool * nkv * page * d * (1 + q.element_size())
    for taken, packed, voting in ((attention, True, 0), (masses, False, votes), (plain_masses, False, votes)):
        assert taken <= ops.compact_cache_workspace(rows, tokens, longest, nq, nkv, d, q.element_size(), packed, voting, sms), (packed, voting, taken)
    ops.raise_on_kernel_errors(torch.device(DEVICE))
