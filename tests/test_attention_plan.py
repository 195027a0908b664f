"""The plan of the document attention, checked on the CPU: every query meets every key it may see exactly once."""

import ctypes
import random

import pytest
import torch

from causal_tuner_b200 import _lib
from causal_tuner_b200.kernels.attention_cuda import KEY_TILE, document_attention, prepare_documents


def documents(rows, width, seed, longest, gap):
    rng, spans = random.Random(seed), []
    for row in range(rows):
        start = rng.randint(0, gap)
        while start < width:
            end = min(width, start + rng.randint(1, longest))
            spans.append((row, start, end))
            start = end + rng.randint(0, gap)
    rng.shuffle(spans)
    return spans


def section(plan, index, records=1):
    first, count = plan.sections[index]
    return plan.table[first:first + count * records].reshape(count, 4 * records).tolist()


@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (4, 1), (32, 1), (24, 8), (3, 1), (256, 2), (128, 1), (16, 16)])
@pytest.mark.parametrize("rows, width, longest, gap", [(1, 1, 1, 0), (2, 700, 600, 0), (3, 501, 200, 30), (1, 3000, 3000, 0), (2, 64, 3, 2)])
def test_plan_covers_every_pair_once(heads, kv_heads, rows, width, longest, gap):
    spans = documents(rows, width, 3, longest, gap)
    plan = prepare_documents((rows, width), spans, "cpu", heads, kv_heads)
    group = heads // kv_heads
    step = _lib.load().ct_attention_tile_tokens(heads, kv_heads)
    assert 128 % step == 0 and group % (128 // step) == 0
    expected = {(row * width + start, end - start) for row, start, end in spans}
    for index, tile in ((0, 2 * step), (1, step), (4, KEY_TILE)):
        seen = {}
        work = []
        for start, length, first, _ in section(plan, index):
            assert (start, length) in expected and 0 <= first < length and first % tile == 0
            assert seen.setdefault(start, set()).isdisjoint({first})
            seen[start].add(first)
            work.append(min(length, first + tile))
        assert all(len(seen[start]) == -(-length // tile) for start, length in expected)
        assert work == sorted(work, reverse=True)
    blocks = group * step // 128
    pieces, slots = {}, set()
    for start, length, key, slot, first, last, _, _ in section(plan, 2, 2):
        assert (start, length) in expected and key % KEY_TILE == 0 and 0 <= key < length and first < last
        pieces.setdefault((start, length, key), []).append((first, last, slot))
        if slot >= 0:
            assert slot not in slots
            slots.add(slot)
    assert slots == set(range(plan.key_slots))
    sums = {token: (rows_, first, count) for token, rows_, first, count in section(plan, 3)}
    assert len(pieces) == sum(-(-length // KEY_TILE) for _, length in expected)
    for (start, length, key), parts in pieces.items():
        parts.sort()
        assert parts[0][0] == 0 and parts[-1][1] == -(-(length - key) // step) * blocks
        assert all(a[1] == b[0] for a, b in zip(parts, parts[1:]))
        if len(parts) == 1:
            assert parts[0][2] == -1 and start + key not in sums
        else:
            count, first, number = sums.pop(start + key)
            assert count == min(KEY_TILE, length - key)
            assert [p[2] for p in parts] == list(range(first, first + number))
    assert not sums
    untouched = set(range(rows * width)) - {t for start, length in expected for t in range(start, start + length)}
    gaps = [t for start, count, _, _ in section(plan, 5) for t in range(start, start + count)]
    assert sorted(gaps) == sorted(untouched) and len(gaps) == len(set(gaps))


def test_refused_spans_and_heads():
    with pytest.raises(ValueError, match="overlap"):
        prepare_documents((1, 10), ((0, 0, 5), (0, 4, 8)), "cpu", 4)
    for span in ((0, -1, 4), (1, 0, 4), (0, 3, 11), (0, 5, 4), (-1, 0, 3)):
        with pytest.raises(ValueError, match="outside"):
            prepare_documents((1, 10), (span,), "cpu", 4)
    for heads, kv_heads in ((4, 3), (0, 1), (4, 0), (2, 4)):
        with pytest.raises(ValueError, match="heads"):
            prepare_documents((1, 10), (), "cpu", heads, kv_heads)
    with pytest.raises(NotImplementedError, match="tokens"):
        prepare_documents((2 ** 16, 2 ** 15), (), "cpu", 4)


def test_plan_entry_point():
    library = _lib.load()
    pair = lambda *values: (ctypes.c_int64 * len(values))(*values)
    sections, slots = (ctypes.c_int64 * 12)(), ctypes.c_int64(-1)

    def plan(starts, lengths, tokens=100, heads=4, kv_heads=1, table=None, capacity=0, sections=sections):
        return library.ct_attention_plan(pair(*starts), pair(*lengths), len(starts), tokens, heads, kv_heads, table, capacity,
                                         sections, ctypes.byref(slots))
    need = plan((50, 0), (50, 40))
    # forward tiles of 64 tokens, query tiles of 32, key pieces (two records), no sums, 128-token tiles, one gap
    assert [sections[i] for i in range(12)] == [0, 2, 2, 4, 6, 2, 10, 0, 10, 2, 12, 1] and need == 13 and slots.value == 0
    table = (ctypes.c_int32 * (4 * need + 4))(*[-7] * (4 * need + 4))
    assert plan((50, 0), (50, 40), table=table, capacity=need) == need
    assert list(table[:8]) == [50, 50, 0, 0, 0, 40, 0, 0] and list(table[48:56]) == [40, 10, 0, 0, -7, -7, -7, -7]
    table = (ctypes.c_int32 * 16)(*[-7] * 16)
    assert plan((50, 0), (50, 40), table=table, capacity=3) == need          # only what fits is written
    assert table[12] == -7
    assert plan((0, 10), (11, 5)) == _lib.ERR_ARG and b"overlap" in library.ct_last_error()
    assert plan((90,), (11,)) == _lib.ERR_ARG and b"outside" in library.ct_last_error()
    assert plan((0,), (-1,)) == _lib.ERR_ARG
    assert plan((0,), (5,), heads=4, kv_heads=3) == _lib.ERR_ARG
    assert plan((0,), (5,), tokens=2 ** 31) == _lib.ERR_UNSUPPORTED
    assert plan((0,), (5,), sections=None) == _lib.ERR_ARG
    assert plan((), (), tokens=0) == 0


def test_no_cpu_path():
    plan = prepare_documents((1, 4), ((0, 0, 4),), "cpu", 2)
    x = torch.zeros(1, 4, 2, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        document_attention(x, x[:, :, :1], x[:, :, :1], plan)


def test_entry_points_check_their_arguments():
    library = _lib.load()
    none = (ctypes.c_int64 * 12)()
    some = (ctypes.c_int64 * 12)(0, 1)
    strides = (None, 64, 64) * 3

    def forward(sections=none, tokens=4, heads=4, kv_heads=1, dim=64, dtype=_lib.BF16, path=_lib.PATH_SIMT):
        return library.ct_attention_forward(*strides, None, None, None, sections, tokens, heads, kv_heads, dim, 1.0, dtype, path, None)

    assert forward(tokens=0) == _lib.OK
    assert forward() == _lib.ERR_ARG
    assert forward(tokens=-1) == _lib.ERR_ARG
    assert forward(kv_heads=3) == _lib.ERR_ARG
    assert forward(dtype=7) == _lib.ERR_ARG
    assert forward(sections=None) == _lib.ERR_ARG
    assert forward(sections=some) == _lib.ERR_ARG and b"plan" in library.ct_last_error()
    assert forward(dim=136) == _lib.ERR_UNSUPPORTED
    assert library.ct_attention_tile_tokens(5, 2) == _lib.ERR_ARG
    assert library.ct_attention_path(*strides, 4, 1, 64, 1.0, 9) == _lib.ERR_ARG
    assert library.ct_attention_path(*strides, 4, 1, 64, 1.0, _lib.F32) == _lib.PATH_SIMT
    # statistics, then the larger of nothing / one fp32 row per head / one 128-row share per slot
    assert library.ct_attention_backward_workspace(100, 4, 4, 64, 0, _lib.PATH_SIMT) == 1792
    assert library.ct_attention_backward_workspace(100, 4, 1, 64, 0, _lib.PATH_SIMT) == 1792 + 2 * 100 * 4 * 64 * 4
