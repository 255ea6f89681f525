"""The paged 4-bit cache without a device: rotation frequencies, what a handle
refuses before it looks for one, and the 64-bit model of the layout."""

import ctypes
import math

import numpy as np
import pytest

import pages_util
from s2hip import PagedKv, S2HipError, _lib, rope_frequencies

GOOD = dict(heads=8, kv_heads=2, head_dim=64, page_tokens=16, pages=10, table_pages=4)


@pytest.mark.parametrize("dims", [2, 16, 64, 128])
def test_plain_frequencies(dims):
    freq, gain = rope_frequencies(dims, 1.0e4)
    assert gain == 1.0 and freq.shape == (dims // 2,)
    np.testing.assert_allclose(freq, [math.exp(-2 * i / dims * math.log(1.0e4)) for i in range(dims // 2)], rtol=1e-14)


def test_scaled_frequencies():
    plain, _ = rope_frequencies(64, 1.0e4)
    line, gain = rope_frequencies(64, 1.0e4, "linear", 4.0)
    np.testing.assert_allclose(line, plain / 4, rtol=1e-15)
    assert gain == 1.0
    stretch, _ = rope_frequencies(64, 1.0e4, "stretch", 4.0)
    assert stretch[0] == 1.0
    np.testing.assert_allclose(stretch[-1], plain[-1] / 4, rtol=1e-13)  # the slowest: all of the factor
    parts, gain = rope_frequencies(64, 1.0e4, "parts", 4.0, context=2048, low=1, high=32)
    assert gain == 1.0 + 0.1 * math.log(4.0)
    for f, was in zip(parts, plain):
        turns = 2048 * was / (2 * math.pi)
        share = min(1.0, max(0.0, (turns - 1) / 31))
        assert abs(f - (was * share + was / 4 * (1 - share))) <= 1e-15 * was
    assert parts[0] == plain[0] and parts[-1] == plain[-1] / 4


@pytest.mark.parametrize("bad, text", [
    (dict(dims=0), "dims"), (dict(dims=7), "dims"), (dict(base=0.0), "base"), (dict(base=math.inf), "base"), (dict(scaling="other"), "scaling"),
    (dict(scaling="linear", factor=0.5), "factor"), (dict(scaling="linear", factor=math.nan), "factor"), (dict(dims=2, scaling="stretch", factor=2.0), "too few"),
    (dict(scaling="parts", factor=2.0, context=0.0), "context"), (dict(scaling="parts", factor=2.0, low=3.0, high=3.0), "low"),
    (dict(scaling="parts", factor=2.0, low=-1.0), "low")])
def test_frequencies_refused(bad, text):
    with pytest.raises(S2HipError, match=text):
        rope_frequencies(**dict(dict(dims=64, base=1.0e4), **bad))


@pytest.mark.parametrize("dims", [-1, -2, -64, -(1 << 31), 1, (1 << 16) + 2, (1 << 32) - 2, (1 << 32) + 64, (1 << 33) + 2])
def test_frequencies_of_impossible_dims(dims):
    """Numbers below 0 and beyond what the C call's 32 bits hold: refused before anything is written."""
    with pytest.raises(S2HipError, match="dims"):
        rope_frequencies(dims, 1.0e4)


@pytest.mark.parametrize("dims", [0, 3, (1 << 16) + 2, (1 << 32) - 2, (1 << 32) - 64])
def test_frequencies_of_impossible_dims_in_c(dims):
    """The C call itself writes to no frequency, whatever a caller's binding makes of its number."""
    L = _lib.load()
    freq, gain, err = np.full(4, 7.0), ctypes.c_double(7.0), ctypes.create_string_buffer(_lib.ERR_CAP)
    assert L.s2hip_rope_frequencies(dims, 1.0e4, 0, 1.0, 8192.0, 1.0, 32.0, freq.ctypes.data, ctypes.byref(gain), err, _lib.ERR_CAP) == 0
    assert b"dims" in err.value and (freq == 7.0).all() and gain.value == 7.0


@pytest.mark.parametrize("bad, text", [
    (dict(heads=0), "heads"), (dict(heads=7), "heads"), (dict(kv_heads=0), "heads"), (dict(heads=130, kv_heads=2), "heads"), (dict(heads=2048, kv_heads=64), "heads"),
    (dict(head_dim=96), "head_dim"), (dict(page_tokens=0), "page_tokens"), (dict(page_tokens=48), "page_tokens"), (dict(page_tokens=256), "page_tokens"),
    (dict(pages=0), "pages"), (dict(pages=(1 << 20) + 1), "pages"), (dict(table_pages=0), "table_pages"), (dict(table_pages=(1 << 16) + 1), "table_pages"),
    (dict(max_requests=0), "max_requests"), (dict(max_requests=257), "max_requests"), (dict(max_tokens=0), "max_tokens"), (dict(max_tokens=65537), "max_tokens"),
    (dict(rope_dims=66), "rope_dims"), (dict(rope_dims=7), "rope_dims"), (dict(rope_dims=24, rope_half=True), "rope_dims"), (dict(rope_base=0.0), "rope_base"),
    (dict(rope_freq=[1.0] * 8, rope_dims=32), "rope_dims"), (dict(rope_freq=[]), "rope_dims"), (dict(rope_freq=[1.0, math.nan]), "rope_freq"),
    (dict(rope_gain=-1.0), "rope_gain"), (dict(eps=-1.0), "eps"), (dict(eps=math.nan), "eps"), (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale")])
def test_handles_refused(bad, text):
    with pytest.raises(S2HipError, match=text):
        PagedKv(**dict(GOOD, **bad))


def test_closed_handle_is_refused():
    ops = PagedKv.__new__(PagedKv)
    import ctypes

    from s2hip import _lib

    ops._h, ops._L, ops._err = None, _lib.load(), ctypes.create_string_buffer(_lib.ERR_CAP)
    view = PagedKv.view(16, 16, 16, 1)
    for call in (lambda: ops.append(view, 16, 1, 16, 16), lambda: ops.attend(view, 16, 1, 16), lambda: ops.update(view, 16, 16, 16, 16),
                 lambda: ops.compact(view, 16, 16, 16, 16), lambda: ops.errors()):
        with pytest.raises(S2HipError, match="NULL"):
            call()
    assert ops.page_bytes == 0


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("hd", [64, 128])
def test_layout_covers_every_bit_once(page, hd):
    lay = pages_util.Layout(page, hd)
    seen = np.zeros(lay.part * 8, int)
    for at, shift in (lay.key, lay.value):
        for bit in range(4):
            np.add.at(seen, (at * 8 + shift + bit).ravel(), 1)
    for at in (lay.key_scale, lay.value_scale):
        for bit in range(16):
            np.add.at(seen, (at * 8 + bit).ravel(), 1)
    assert (seen == 1).all()


def test_every_element_is_an_f16_number():
    """The scale's 8 significant bits times a code's 4 fit the 11 of an f16, to the ends of its range."""
    for top in [16383.9, 10000.0, 3.0, 1.0 + 2.0**-9, 2.0**-13 * 1.37, 2.0**-20 * 1.9, 2.0**-22, 2.0**-23, 0.0]:
        x = np.linspace(-1, 1, 32) * top
        code, d, held = pages_util.quantised(x)
        assert (held.astype(np.float16).astype(np.float64) == held).all() and (d.astype(np.float16).astype(np.float64) == d).all()
        if top <= 2.0**-22:  # an eighth of it is at most half of 2^-24, which rounds to 0
            assert (held == 0).all() and (d == 0).all()
            continue
        step = abs(d[0]) * 0.5 * (1 + 2.0**-8) + 2.0**-25
        clipped = (code == 15) | (code == 0)
        assert (np.abs(held - x) <= np.where(clipped, abs(d[0]) * (1 + 2.0**-4), step)).all()
