"""Calls of the paged cache and of the logits that are refused, without a GPU: arguments are
checked before anything else."""
import ctypes as C

import numpy as np
import pytest

import mojostream_amd as ms

INVALID, STATE = -1, -3


def err():
    return ms.lib().ms_last_error().decode()


@pytest.mark.parametrize("sizes", [(0, 4, 1, 1, 1), (16, 0, 1, 1, 1), (16, 4, 0, 1, 1), (16, 4, 1, 0, 1),
                                   (16, 4, 1, 1, 0), (1 << 16, 1 << 15, 1, 1, 1), (1 << 20, 4, 1, 1, 1 << 11)])
def test_batch_sizes(sizes):
    h = C.c_void_p(1)
    assert ms.lib().ms_paged_batch_create(*sizes, C.byref(h)) == INVALID
    assert h.value is None


@pytest.fixture()
def batch():
    b = ms.PagedBatch(4, 10, 3, 20, 5)
    yield b
    b.close()


def _set(b, new, length, pages):
    n, l = np.array(new, np.int32), np.array(length, np.int32)
    p = np.full((max(len(new), 1), 5), -9, np.int32)
    for s, row in enumerate(pages):
        p[s, :len(row)] = row
    return ms.lib().ms_paged_batch_set(b.h, len(new), n.ctypes.data, l.ctypes.data, p.ctypes.data)


@pytest.mark.parametrize("new,length,pages,say", [
    ([1], [0], [[0]], "less than its new rows"),
    ([-1], [4], [[0]], "less than its new rows"),
    ([1], [21], [[0, 1, 2, 3, 4]], "more positions than its pages"),
    ([1], [5], [[0, 10]], "page 1 is 10"),
    ([1], [5], [[0, -2]], "page 1 is -2"),
    ([1], [9], [[0, -1, 2]], "page 1 is -1"),
    ([1], [5], [[0, -1]], "page 1 is -1"),
    ([1], [5], [[-1, -1]], "a new row's page is missing"),
    ([5], [9], [[-1, -1, 2]], "a new row's page is missing"),
    ([1, 1], [4, 4], [[3], [3]], "page 3 would be written twice"),
    ([8], [8], [[3, 3]], "page 3 would be written twice"),
    ([10, 11], [10, 11], [[0, 1, 2], [3, 4, 5]], "more rows than the batch holds"),
    ([1] * 4, [1] * 4, [[0], [1], [2]], "too many sequences"),
])
def test_batch_set(batch, new, length, pages, say):
    if len(new) > 3:
        pages = pages + [[3]]
    assert _set(batch, new, length, pages) == INVALID
    assert say in err(), err()


@pytest.mark.parametrize("new,length,pages", [
    ([1], [1], [[9]]),
    ([0], [0], [[]]),
    ([1], [13], [[-1, -1, -1, 7]]),               # freed behind a window
    ([1, 1], [6, 7], [[0, 1], [0, 2]]),           # a shared prefix
    ([4, 0], [4, 4], [[0], [0]]),                 # read by one, written by another
    ([], [], []),
])
def test_batch_set_needs_init(batch, new, length, pages):
    """What may be set gets as far as the missing GPU."""
    if ms.lib().ms_synchronize() == 0:
        pytest.skip("a GPU is in use")
    assert _set(batch, new, length, pages) == STATE


def test_batch_null(batch):
    assert ms.lib().ms_paged_batch_set(None, 0, None, None, None) == INVALID
    assert ms.lib().ms_paged_batch_set(batch.h, 1, None, None, None) == INVALID
    with pytest.raises(ms.MSError):
        batch.set([1], [1], np.zeros((1, 6), np.int32))
    with pytest.raises(ms.MSError):
        batch.set([1], [1, 2], np.zeros((1, 5), np.int32))


@pytest.mark.parametrize("new,length,pages", [
    ([1], [1], [[2 ** 32 + 3]]), ([2 ** 32 + 1], [2 ** 32 + 1], [[3]]), ([1], [2 ** 32 + 1], [[3]]),
    ([1], [1], [[1.5]]), ([0.5], [1], [[3]]), ([1], [float("nan")], [[3]]), ([1], [2 ** 70], [[3]])])
def test_set_takes_int32_values(batch, new, length, pages):
    """Numbers that 32 bits do not hold are refused, not wrapped to others."""
    with pytest.raises(ms.MSError, match="32-bit"):
        batch.set(np.array(new), np.array(length), np.array(pages))


GOOD = dict(n_heads=8, n_kv_heads=2, head_dim=64, rot_dim=64, window=0, dtype=0, page_rows=0, scale=0.0,
            k=4096, v=8192)


@pytest.mark.parametrize("change,say", [
    (dict(n_heads=7), "multiple of n_kv_heads"), (dict(n_kv_heads=0), "multiple of n_kv_heads"),
    (dict(head_dim=96), "head_dim"), (dict(dtype=3), "pool type"), (dict(window=-1), "window"),
    (dict(page_rows=3), "page_rows"), (dict(page_rows=1 << 28), "2^31 rows"), (dict(k=None), "null pool"),
    (dict(v=8200), "aligned"), (dict(n_heads=2048), "1024"), ({}, "was not set")])
def test_layers(batch, change, say):
    layer = ms.PagedLayer(**{**GOOD, **change})
    for call in (lambda: ms.lib().ms_paged_attention(C.byref(layer), batch.h, 4096, 512, 8192, 512),
                 lambda: ms.lib().ms_paged_append(C.byref(layer), batch.h, 4096, 4096, 128, 4096, 512, 4096, 512,
                                                  4096, 4096, 100)):
        assert call() == INVALID
        assert say in err(), err()


def test_layer_arguments(batch):
    for change in (dict(rot_dim=3), dict(rot_dim=66), dict(rot_dim=-2)):
        layer = ms.PagedLayer(**{**GOOD, **change})
        assert ms.lib().ms_paged_append(C.byref(layer), batch.h, 0, 0, 128, 0, 0, 0, 0, 64, 64, 9) == INVALID
        assert "rot_dim" in err()
    layer = ms.PagedLayer(**GOOD)
    assert ms.lib().ms_paged_append(C.byref(layer), batch.h, 64, 64, 128, 0, 0, 0, 0, None, 64, 9) == INVALID
    assert "tables" in err()
    for scale in (float("nan"), float("inf")):
        layer = ms.PagedLayer(**{**GOOD, "scale": scale})
        assert ms.lib().ms_paged_attention(C.byref(layer), batch.h, 64, 512, 64, 512) == INVALID
        assert "scale" in err()
    assert ms.lib().ms_paged_attention(None, batch.h, 64, 512, 64, 512) == INVALID
    assert ms.lib().ms_paged_append(C.byref(ms.PagedLayer(**GOOD)), None, 64, 64, 128, 0, 0, 0, 0, 64, 64, 9) == INVALID


@pytest.mark.parametrize("args", [(None, 64, 64, 1e4, 0, 8), (64, None, 64, 1e4, 0, 8), (64, 64, 63, 1e4, 0, 8),
                                  (64, 64, 0, 1e4, 0, 8), (64, 64, 64, -1.0, 0, 8), (64, 64, 64, float("nan"), 0, 8),
                                  (64, 64, 64, 1e4, -1, 8), (64, 64, 64, 1e4, 0, -1), (64, 64, 64, 1e4, 2 ** 31 - 1, 8)])
@pytest.mark.parametrize("wide", [0, 1])
def test_rope_table(args, wide):
    assert ms.lib().ms_rope_table(*args, wide) == INVALID


@pytest.mark.parametrize("wide", [0, 1])
def test_rope_table_size(wide):
    assert ms.lib().ms_rope_table(64, 64, 64, 1e4, 0, 2 ** 26 + 1, wide) == INVALID
    assert "too large" in err()


@pytest.mark.parametrize("scale", [2.4e38, -3.4e38])
def test_scale_past_fp32_in_log2(batch, scale):
    layer = ms.PagedLayer(**{**GOOD, "scale": scale})
    assert ms.lib().ms_paged_attention(C.byref(layer), batch.h, 64, 512, 64, 512) == INVALID
    assert "scale" in err()


def _logits(row=None, n=1, vocab=100, x=4096, ldx=100, y=8192, ldy=100, hist=64, nh=10, ids=64, vals=64, nb=5,
            masks=64, nm=2):
    rows = (ms.LogitsRow * max(n, 1))(*[row or ms.LogitsRow()] * max(n, 1))
    return ms.lib().ms_logits_process(x, ldx, y, ldy, n, vocab, rows, hist, nh, ids, vals, nb, masks, nm)


@pytest.mark.parametrize("row,say", [
    (dict(repetition=0.0), "repetition"), (dict(repetition=-1.0), "repetition"),
    (dict(repetition=float("nan")), "repetition"), (dict(repetition=float("inf")), "repetition"),
    (dict(frequency=float("nan")), "penalty"), (dict(presence=float("-inf")), "penalty"),
    (dict(n_prompt=-1), "negative"), (dict(n_generated=-1), "negative"), (dict(n_bias=-1), "negative"),
    (dict(history=-1, n_prompt=1), "history"), (dict(history=6, n_prompt=2, n_generated=3), "history"),
    (dict(history=11), "history"), (dict(history=2 ** 62, n_prompt=2 ** 30), "history"),
    (dict(n_prompt=2 ** 31 - 1, n_generated=2 ** 31 - 1), "history"),
    (dict(bias=3, n_bias=3), "biases"), (dict(bias=-1), "biases"),
    (dict(mask=2), "mask"), (dict(mask=-2), "mask")])
def test_logits_rows(row, say):
    assert _logits(ms.LogitsRow(**row)) == INVALID
    assert "row 0" in err() and say in err(), err()


@pytest.mark.parametrize("row,say", [(dict(n_bias=2 ** 30), "biases"), (dict(n_bias=2 ** 31 - 1), "biases"),
                                     (dict(n_prompt=2 ** 30), "history"),
                                     (dict(n_prompt=2 ** 30 - 1, n_generated=1), "history")])
def test_logits_counts(row, say):
    """Counts that the kernel's 32-bit indexes do not hold, over arrays that would be large enough."""
    assert _logits(ms.LogitsRow(**row), hist=64, nh=2 ** 33, nb=2 ** 33) == INVALID
    assert "row 0" in err() and say in err(), err()


def test_logits_arguments():
    assert _logits(n=-1) == INVALID
    assert _logits(vocab=0) == INVALID
    assert _logits(x=None) == INVALID
    assert _logits(y=None) == INVALID
    assert _logits(ldx=99) == INVALID
    assert _logits(ldy=99) == INVALID
    assert _logits(nm=-1) == INVALID
    assert _logits(y=4096 + 4, n=2) == INVALID and "overlap" in err()
    assert _logits(y=4096, n=2, ldy=101) == INVALID and "overlap" in err()
    assert _logits(ms.LogitsRow(n_prompt=1), hist=None) == INVALID
    assert _logits(ms.LogitsRow(n_bias=1), vals=None) == INVALID
    assert _logits(ms.LogitsRow(mask=0), masks=None) == INVALID
    if ms.lib().ms_synchronize() != 0:
        assert _logits() == STATE and _logits(n=0) == STATE
        assert _logits(y=4096) == STATE               # in place
        assert _logits(y=4096 + 400, ldx=200, ldy=200, n=3) == STATE  # rows beside each other
