"""8-bit attention refuses an out that overlaps q otherwise than as q itself: at the C entry, on the CPU."""

from __future__ import annotations

import ctypes

import pytest

from plastic_infer import _native as N

ROW = 4 * 16 * 2      # bytes of a row: 4 heads of 16, bf16


def _call(out, q, stride, rows):
    """(refused as overlapping, where it stopped) of a call that has everything but a workspace's size."""
    buf = ctypes.create_string_buffer(4096)
    base = (ctypes.addressof(buf) + 255) // 256 * 256
    lib = N.load()
    rc = lib.pia_kv8_attention(base + out, base + q, stride, base, base, base, base, base, 1, base,
                               None, None, rows, rows, 4, 2, 16, 16, 4, 1.0, 2, base, 0, None)
    assert rc == -1
    return "overlaps" in lib.pia_last_error().decode()


@pytest.mark.parametrize("out,q,stride,rows,bad", [
    (0, 0, 64, 3, False), (0, 3 * ROW, 64, 3, False), (3 * ROW, 0, 64, 3, False),
    (0, 3 * ROW - 16, 64, 3, True), (3 * ROW - 16, 0, 64, 3, True), (16, 0, 64, 3, True),
    (0, 16, 64, 3, True), (0, 0, 128, 3, True), (0, 0, 64, 1, False),
    (ROW, 0, 64, 1, False), (ROW, 0, 640, 3, False),          # between two rows of a wide q
    (ROW, 0, 192, 3, True), (10 * ROW - 16, 0, 640, 3, True), (21 * ROW, 0, 640, 3, False),
    (21 * ROW - 16, 0, 640, 3, True), (0, 0, 0, 3, True), (ROW, 0, 0, 3, False)])
def test_overlap(out, q, stride, rows, bad):
    assert _call(out, q, stride, rows) == bad
