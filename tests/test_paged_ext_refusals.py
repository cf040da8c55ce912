"""Calls of the 8-bit cache, the normed append, the capped attention and the row sampler that are refused, without
a GPU: arguments are checked before anything else."""
import ctypes as C

import numpy as np
import pytest

import mojostream_amd as ms
from tests.paged_ext_ref import E4M3, nearest, scale_of

INVALID, STATE = -1, -3


def err():
    return ms.lib().ms_last_error().decode()


@pytest.fixture()
def batch():
    b = ms.PagedBatch(4, 10, 3, 20, 5)
    yield b
    b.close()


BASE = dict(n_heads=8, n_kv_heads=2, head_dim=64, rot_dim=64, window=0, dtype=4, page_rows=0, scale=0.0, k=4096, v=8192)
EXT = dict(k_scale=4096, v_scale=8192)


def layer(**change):
    base = {**BASE, **{k: v for k, v in change.items() if k in BASE}}
    return ms.PagedLayerExt(base=ms.PagedLayer(**base), **{**EXT, **{k: v for k, v in change.items() if k not in BASE}})


def attend(L, b, q=4096, out=1 << 20):
    return ms.lib().ms_paged_attention_ext(C.byref(L), b.h if b else None, q, 512, out, 512)


def append(L, b):
    return ms.lib().ms_paged_append_ext(C.byref(L), b.h if b else None, 4096, 4096, 128, 4096, 512, 4096, 512, 4096,
                                        4096, 100)


def read(L, b):
    return ms.lib().ms_paged_read(C.byref(L), b.h if b else None, 0, 0, 1, 4096, None, 128)


@pytest.mark.parametrize("change,say", [
    (dict(n_heads=7), "multiple of n_kv_heads"), (dict(head_dim=96), "head_dim"), (dict(dtype=3), "pool type"),
    (dict(dtype=6), "pool type"), (dict(dtype=-1), "pool type"), (dict(window=-1), "window"),
    (dict(page_rows=3), "page_rows"), (dict(k=None), "null pool"), (dict(v=8200), "aligned"),
    (dict(k_scale=None), "has scales"), (dict(dtype=5, v_scale=None), "has scales"), (dict(v_scale=4097), "scales must be"),
    ({}, "was not set"), (dict(dtype=0, k_scale=None, v_scale=None), "was not set")])
def test_layers(batch, change, say):
    L = layer(**change)
    for call in (attend, append, read):
        assert call(L, batch) == INVALID
        assert say in err(), err()


@pytest.mark.parametrize("cap,scale,ok", [
    (float("nan"), 0.0, False), (float("inf"), 0.0, False), (-1.0, 0.0, False), (2.0 ** -61, 0.0, False), (2.0 ** 61, 0.0, False),
    (2.0 ** -60, 2.0 ** 70, False), (2.0 ** 60, 2.0 ** -70, False), (30.0, float("nan"), False), (30.0, float("inf"), False),
    (2.0 ** -60, 2.0 ** 60, True), (2.0 ** 60, -(2.0 ** -60), True), (0.0, 2.0 ** -100, True)])
def test_caps(batch, cap, scale, ok):
    assert attend(layer(score_cap=cap, scale=scale), batch) == INVALID
    assert ("was not set" in err()) == ok and (ok or "scale" in err() or "score_cap" in err()), err()


@pytest.mark.parametrize("change,say", [
    (dict(norm=8), "unknown norm"), (dict(norm=-1), "unknown norm"), (dict(norm=1, norm_eps=-1e-9), "norm_eps"),
    (dict(norm=2, norm_eps=float("nan")), "norm_eps"), (dict(norm=4, norm_eps=float("inf")), "norm_eps"),
    (dict(rope=2), "unknown rotation"), (dict(rope=-1), "unknown rotation"), (dict(q_gamma=4098), "gammas"),
    (dict(k_gamma=4099), "gammas"), (dict(norm=7, norm_eps=0.0, rope=1, q_gamma=4100, k_gamma=4100), "was not set")])
def test_norms_and_rotations(batch, change, say):
    assert append(layer(**change), batch) == INVALID
    assert say in err(), err()


def test_null(batch):
    L = layer()
    for call in (attend, append, read):
        assert call(L, None) == INVALID
    lib = ms.lib()
    assert lib.ms_paged_attention_ext(None, batch.h, 4096, 512, 8192, 512) == INVALID
    assert lib.ms_paged_append_ext(None, batch.h, 4096, 4096, 128, None, 0, None, 0, None, None, 0) == INVALID
    assert lib.ms_paged_read(None, batch.h, 0, 0, 0, None, None, 0) == INVALID


@pytest.mark.parametrize("dtype", [4, 5])
def test_the_plain_calls_refuse_8_bits(batch, dtype):
    L = ms.PagedLayer(**{**BASE, "dtype": dtype})
    assert ms.lib().ms_paged_attention(C.byref(L), batch.h, 4096, 512, 8192, 512) == INVALID and "pool type" in err()
    assert ms.lib().ms_paged_append(C.byref(L), batch.h, 4096, 4096, 128, None, 0, None, 0, 4096, 4096, 9) == INVALID
    assert "pool type" in err()


ROW = dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0)


@pytest.mark.parametrize("change,say", [
    (dict(temperature=-0.1), "temperature"), (dict(temperature=float("inf")), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(top_k=-1), "top_k"), (dict(top_p=-0.1), "top_p"),
    (dict(top_p=1.1), "top_p"), (dict(top_p=float("nan")), "top_p"), (dict(min_p=-1e-9), "min_p"),
    (dict(min_p=1.001), "min_p"), (dict(min_p=float("nan")), "min_p")])
def test_sample_settings(change, say):
    rows = (ms.SampleRow * 2)(ms.SampleRow(), ms.SampleRow(**{**ROW, **change}))
    assert ms.lib().ms_sample_rows(4096, 100, 2, 100, rows, 4096, 4096, None, None) == INVALID
    assert say in err() and "row 1" in err(), err()


@pytest.mark.parametrize("x,ld,n,v,u,ids", [(None, 100, 1, 100, 4096, 4096), (4096, 99, 1, 100, 4096, 4096),
                                            (4096, 100, -1, 100, 4096, 4096), (4096, 100, 1, 0, 4096, 4096),
                                            (4096, 1 << 31, 1, (1 << 30) + 1, 4096, 4096),
                                            (4096, 100, 1, 100, None, 4096), (4096, 100, 1, 100, 4096, None),
                                            (4096, 1 << 41, 1, 100, 4096, 4096)])
def test_sample_arguments(x, ld, n, v, u, ids):
    rows = (ms.SampleRow * 1)(ms.SampleRow())
    assert ms.lib().ms_sample_rows(x, ld, n, v, rows, u, ids, None, None) == INVALID
    assert ms.lib().ms_sample_rows(4096, 100, 1, 100, None, 4096, 4096, None, None) == INVALID


def test_good_arguments_need_init():
    if ms.lib().ms_synchronize() == 0:
        pytest.skip("a GPU is in use")
    rows = (ms.SampleRow * 1)(ms.SampleRow())
    assert ms.lib().ms_sample_rows(4096, 100, 1, 100, rows, 4096, 4096, None, None) == STATE
    assert ms.lib().ms_sample_rows(4096, 100, 0, 100, None, None, None, None, None) == STATE


def test_the_tests_own_codes():
    """The e4m3 table and the rounding that the GPU tests compare with, by hand."""
    assert E4M3[0x08] == 2.0 ** -6 and E4M3[0x01] == 2.0 ** -9 and E4M3[0x7E] == 448 and E4M3[0x38] == 1
    assert np.isnan(E4M3[0x7F]) and E4M3[0xB8] == -1 and np.all(np.diff(E4M3[:127]) > 0)
    c, near = nearest(np.array([1.0625, 1.1875, 1.0626, -1.0625, 2.0 ** -10, 3 * 2.0 ** -10, 448.4, 0.0]), "e4m3")
    assert E4M3[c].tolist() == [1.0, 1.25, 1.125, -1.0, 0.0, 2.0 ** -8, 448.0, 0.0] and not near.any()
    c, _ = nearest(np.array([0.5, 1.5, -2.5, 126.6]), "i8")
    assert c.view(np.int8).tolist() == [0, 2, -2, 127]
    assert scale_of(np.array([[0.0, 0], [896, 1], [np.inf, 1], [np.nan, 1]]), "e4m3").tolist()[:2] == [2.0 ** -126, 2.0]
    assert np.isnan(scale_of(np.array([[np.inf, 1], [np.nan, 1]]), "i8")).all()
