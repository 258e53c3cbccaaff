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


# ---------------------------------------------------------------------------------------
# decoded tokens over the codes: values and scores of unlike sizes
# ---------------------------------------------------------------------------------------
def pages_of(rows, page, group):
    """4-bit pages that hold ``rows [slots, nkv, d]`` one page after another, and their table."""
    from pylon_b200.kernels import ops

    slots, nkv, d = rows.shape
    count = -(-slots // page)
    full = torch.zeros(count * page, nkv, d, dtype=torch.float64, device=DEVICE)
    full[:slots] = rows
    return ops.PackedPages(*plain.pack(full.view(count, page, nkv, d).transpose(1, 2), group)), torch.arange(count, dtype=torch.int32, device=DEVICE)[None]


def decoded(q, keys, values, group, page=64, scale=None):
    """One bfloat16 token over ``keys`` and ``values [slots, nkv, d]``: the result, the result in 64 bits, the sum of the weights times the values' sizes, every channel's
    rounding of weights (float16, times the step) and of scores (codes as subnormal numbers), as bounds."""
    from pylon_b200.kernels import ops

    slots, nkv, d = keys.shape
    nq = q.shape[1] // d
    scale = d ** -0.5 if scale is None else scale
    k_pages, table = pages_of(keys, page, group)
    v_pages, _ = pages_of(values, page, group)
    got = ops.paged_attention_packed(q, k_pages, v_pages, ints([slots - 1]), ints([0]), ints([0, 1]), ints([slots]), table, nq, 1, slots, scale=scale)
    ops.raise_on_kernel_errors(torch.device(DEVICE))
    expected, size = plain.attention(q, k_pages, v_pages, [1], [slots], table, nq, scale)
    largest = plain.steps(v_pages.words).amax((0, 2)).repeat_interleave(group, -1)                      # [nkv, d]: every group's largest step
    terms = slots * 2.0 ** -27 * largest.repeat_interleave(nq // nkv, 0).flatten()
    most = q.double().abs().view(nkv, nq // nkv, d).amax(1).unflatten(-1, (-1, group)).amax(-1)           # [nkv, groups]
    score = scale * 15 * 2.0 ** -14 * float((plain.steps(k_pages.words).amax((0, 2)) * most).sum(-1).max())
    share = 2.0 ** -11 + 2 * score + 4 * (d + 4) * 2.0 ** -24 * scale * float(torch.linalg.vector_norm(q.double().view(-1, d), dim=-1).max() * torch.linalg.vector_norm(keys, dim=-1).max())
    return got.double(), expected, size, HALF[torch.bfloat16] * expected.abs() + share * size + terms


@pytest.mark.parametrize("slots", [40, 700, 5000])
@pytest.mark.parametrize("d, group", [(128, 32), (128, 64), (64, 32)])
@pytest.mark.parametrize("apart", [0, 16, -16, 28, -28, 60])
def test_groups_of_values_of_unlike_size(apart, d, group, slots):
    """Every group is right by its own measure, however much larger the others are."""
    nq, nkv = 8, 2
    values = torch.randn(slots, nkv, d, dtype=torch.float64, device=DEVICE)
    values[..., group:] *= 2.0 ** apart
    q = torch.randn(1, nq * d, device=DEVICE).bfloat16()
    got, expected, size, bound = decoded(q, torch.randn(slots, nkv, d, dtype=torch.float64, device=DEVICE), values, group)
    assert ((got - expected).abs() <= bound).all(), float(((got - expected).abs() / size).max())


@pytest.mark.parametrize("d, group", [(128, 32), (128, 64), (64, 32)])
@pytest.mark.parametrize("apart", [20, -20, 40])
@pytest.mark.parametrize("seen", [True, False])
def test_a_late_key_whose_groups_are_of_unlike_size(seen, apart, d, group):
    """A key far into the context whose first group alone is much larger (or all others are), seen or passed over: the other groups keep what they had."""
    nq, nkv, slots = 8, 2, 3000
    keys, values = (torch.randn(slots, nkv, d, dtype=torch.float64, device=DEVICE) for _ in range(2))
    q = torch.randn(1, nq * d, device=DEVICE).bfloat16()
    if not seen:      # its score is far below the others'
        keys[2500] = -8 * q.double().view(nkv, nq // nkv, d).mean(1)
    if apart > 0:
        values[2500, :, :group] *= 2.0 ** apart
    else:
        values[2500, :, group:] *= 2.0 ** -apart
    got, expected, size, bound = decoded(q, keys, values, group)
    assert ((got - expected).abs() <= bound).all(), float(((got - expected).abs() / size).max())


@pytest.mark.parametrize("d, group", [(128, 128), (128, 32), (64, 64)])
@pytest.mark.parametrize("below, slots", [(10.0, 5_000), (16.6, 100_000), (18.0, 200_000)])
def test_many_small_weights_beside_one(below, slots, d, group):
    """One key far above a long flat context: the others' weights, e^-below each, still count where that key has no value."""
    nq, nkv = 2, 1
    keys, values = torch.zeros(slots, nkv, d, dtype=torch.float64, device=DEVICE), torch.ones(slots, nkv, d, dtype=torch.float64, device=DEVICE)
    keys[slots // 3, :, 0] = below / 4
    values[slots // 3] = 0.0
    q = torch.zeros(1, nq * d, device=DEVICE).bfloat16()
    q[:, ::d] = 4.0
    got, expected, size, bound = decoded(q, keys, values, group, scale=1.0)
    assert ((got - expected).abs() <= bound).all() and (bound <= 0.05 * expected).all(), (float(got.max()), float(expected.max()))


@pytest.mark.parametrize("d, group", [(128, 128), (128, 64), (128, 32), (64, 64)])
def test_scores_that_are_differences_of_large_sums(d, group):
    """Queries of one sign over keys whose codes lie around the middle: the product over the codes is far larger than the score that is left of it.  A score is off by 2^-14 of
    15 steps times the largest query, group by group."""
    nq, nkv, slots = 8, 2, 300
    keys = torch.randn(slots, nkv, d, dtype=torch.float64, device=DEVICE)
    q = (3.0 + torch.rand(1, nq * d, device=DEVICE)).bfloat16()
    got, expected, size, bound = decoded(q, keys * 0.05, torch.randn(slots, nkv, d, dtype=torch.float64, device=DEVICE), group, scale=1.0)
    assert ((got - expected).abs() <= bound).all(), float(((got - expected).abs() / size).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d, nq", [(128, 8), (64, 40), (96, 8)])
def test_a_single_query_anywhere_in_memory(d, nq, dtype):
    """One token's row counts as contiguous whatever its stride and its address."""
    from pylon_b200.kernels import ops

    nkv, page, counts, lengths = 2, 16, [1], [70]
    table, pool, q_start, kv_len, row, slots = tables(counts, lengths, page)
    k_pages, v_pages = random_pages(pool, nkv, page, d, 32), random_pages(pool, nkv, page, d, 32)
    row_of = torch.randn(1, nq * d + 5, device=DEVICE).to(dtype)
    results = []
    for q in (row_of[:, :-5], row_of[:, 3:-2], row_of):
        got = ops.paged_attention_packed(q, k_pages, v_pages, slots, row, q_start, kv_len, table, nq, 1, 70)
        aligned = torch.empty(1, nq * d, dtype=dtype, device=DEVICE).copy_(q[:, : nq * d])
        assert torch.equal(got, ops.paged_attention_packed(aligned, k_pages, v_pages, slots, row, q_start, kv_len, table, nq, 1, 70))
        mass, other = torch.zeros(pool, nkv, page, device=DEVICE), torch.zeros(pool, nkv, page, device=DEVICE)
        ops.attention_mass(q, k_pages, mass, q_start, kv_len, table, nq, 1, 70)
        ops.attention_mass(aligned, k_pages, other, q_start, kv_len, table, nq, 1, 70)
        torch.testing.assert_close(mass, other, rtol=1e-4, atol=1e-6)      # (scores in 32 bits, on another kernel where the row is off its alignment)
        results.append(got)
    ops.raise_on_kernel_errors(torch.device(DEVICE))
