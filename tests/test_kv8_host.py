"""What the entry points over caches of 8 bits refuse, ahead of any launch (include/bitnet_hip.h section 5: kv8_*), and the order of their values, restated two ways.  No GPU."""
import importlib
import os

import numpy as np
import pytest

from tests import kv8_util as kv


@pytest.fixture(scope="module")
def built(pkg):
    if not os.path.exists(pkg.LIB_PATH):
        pkg.build()
    return importlib.import_module("bitnet-rs_amd")


def test_refusals(built):
    hip = built.load()

    def gqa(heads=4, kv_heads=2, maps=1, dim=16, dimp=32, vdim=16, vdimp=32, capacity=128, k=16, v=16, **more):
        return built.Gqa(heads, kv_heads, maps, dim, dimp, vdim, vdimp, capacity, 1e-5, 0.1, 0.9, 8, 8, 8, k, v, **more)

    g, wide = gqa(), gqa(dim=288, dimp=288, vdim=288, vdimp=288)
    bad = [
        (lambda: hip.kv8_rows_dev(gqa(kv_heads=3), 16, 16, 16, 256, True, 8, 1), "gqa: bad shape"),
        (lambda: hip.kv8_rows_dev(gqa(capacity=100), 16, 16, 16, 256, True, 8, 1), "gqa: bad shape"),
        (lambda: hip.kv8_rows_dev(wide, 16, 16, 16, 4096, True, 8, 1), "kv8: head of 288 / 288 columns"),
        (lambda: hip.kv8_rows_dev(g, 24, 16, 16, 256, True, 8, 1), "16 bytes"),
        (lambda: hip.kv8_rows_dev(gqa(k=24), 16, 16, 16, 256, True, 8, 1), "16 bytes"),
        (lambda: hip.kv8_rows_dev(g, 0, 16, 16, 256, True, 8, 1), "16 bytes"),
        (lambda: hip.kv8_rows_dev(g, 16, 16, 16, 255, True, 8, 1), "kv8_rows: bad arguments"),
        (lambda: hip.kv8_rows_dev(g, 16, 16, 16, 256, True, 8, 0), "kv8_rows: bad arguments"),
        (lambda: hip.kv8_rows_dev(g, 16, 16, 16, 260, True, 8, 2), "kv8_rows: bad arguments"),
        (lambda: hip.kv8_rows_dev(g, 16, 16, 24, 256, True, 8, 2), "kv8_rows: bad arguments"),
        (lambda: hip.kv8_rows_dev(g, 16, 16, 16, 256, True, 8, 129), "kv8_rows: bad arguments"),
        (lambda: hip.kv8_rows_dev(g, 16, 16, 16, 256, True, 0, 1), "kv8_rows: bad arguments"),
        (lambda: hip.kv8_rows_dev(g, 16, 16, 16, 256, True, 8, 1, 32, 127), "place of the queries"),
        (lambda: hip.kv8_rows_dev(g, 16, 16, 16, 256, True, 8, 1, 16, 128), "place of the queries"),
        (lambda: hip.kv8_rows_dev(gqa(taps=3, conv=8, ring=8), 16, 16, 16, 256, True, 8, 2), "place of the queries"),
        (lambda: hip.kv8_read_dev(g, 16, 16, 0, 0, 16, 16, True), "kv8_read"),
        (lambda: hip.kv8_read_dev(g, 16, 16, 1, 128, 16, 16, True), "kv8_read"),
        (lambda: hip.kv8_read_dev(g, 16, 16, 2 ** 64 - 1, 2, 16, 16, True), "kv8_read"),
        (lambda: hip.kv8_read_dev(g, 16, 16, 0, 1, None, None, True), "kv8_read"),
        (lambda: hip.kv8_read_dev(g, 16, 16, 0, 1, 24, None, True), "kv8_read"),
        (lambda: hip.kv8_step_dev(g, 16, 16, 0, 8, 16), "kv8_step"),
        (lambda: hip.kv8_step_dev(g, 16, 16, 16, 8, 24), "kv8_step"),
        (lambda: hip.kv8_step_dev(wide, 16, 16, 16, 8, 16), "kv8: head"),
        (lambda: hip.kv8_step_dev(gqa(maps=2, sink=8), 16, 16, 16, 8, 16), "gqa: bad chunk, sink"),
        (lambda: hip.kv8_prefill_dev(g, 16, 16, 16, 128, 10, 11, 16, 128), "kv8_prefill: bad arguments"),
        (lambda: hip.kv8_prefill_dev(g, 16, 16, 16, 128, 129, 11, 16, 128), "kv8_prefill: bad arguments"),
        (lambda: hip.kv8_prefill_dev(g, 16, 16, 16, 120, 10, 10, 16, 128), "kv8_prefill: bad arguments"),
        (lambda: hip.kv8_prefill_dev(g, 16, 16, 16, 132, 10, 10, 16, 128), "kv8_prefill: bad arguments"),
        (lambda: hip.kv8_prefill_dev(g, 16, 16, 24, 128, 10, 10, 16, 128), "kv8_prefill: bad arguments"),
        (lambda: hip.kv8_prefill_dev(g, 16, 16, 16, 128, 10, 10, 16, 126), "kv8_prefill: bad arguments"),
        (lambda: hip.kv8_prefill_dev(gqa(capacity=4096), 16, 16, 16, 128, 4000, 10, 16, 128, 16, 16), "kv8_prefill: scratch of 16 bytes"),
        (lambda: hip.kv8_prefill_dev(gqa(maps=2, dim=160, dimp=160), 16, 16, 16, 1280, 10, 10, 16, 128), "want scratch"),
        (lambda: hip.kv8_prefill_dev(wide, 16, 16, 16, 2048, 10, 10, 16, 2048), "kv8: head"),
    ]
    for i, (call, match) in enumerate(bad):
        with pytest.raises(built.BitNetHipError, match=match):
            call()
            pytest.fail(str(i))
    assert hip.kv8_prefill_scratch_bytes(wide, 10, 10) == 0 and hip.kv8_prefill_scratch_bytes(g, 10, 11) == 0 and hip.kv8_prefill_scratch_bytes(gqa(capacity=4096), 4000, 10) > 0


def test_order_of_the_values():
    g, p, v = 2, 128, 96
    x = np.random.default_rng(0).integers(-127, 128, (g, p, v)).astype(np.int8)
    packed = kv.pack(x)
    assert packed.shape == (g, p // 32, v // 32, 16, 4, 2, 8) and np.array_equal(kv.unpack(packed), x)
    pos, col = np.meshgrid(np.arange(p), np.arange(v), indexing="ij")
    assert np.array_equal(packed[:, pos // 32, col // 32, col % 16, pos % 32 // 8, col % 32 // 16, pos % 8], x)


def test_numbers_of_a_vector():
    n, s = kv.numbers_of([[1.0, -2.0, 0.5, 0.0], [0, 0, 0, 0], [np.nan, 1, 2, 3], [127, 0.5, 1.5, -2.5]])
    assert n.tolist() == [[64, -127, 32, 0], [0, 0, 0, 0], [0, 0, 0, 0], [127, 0, 2, -2]] and s[1] == 0 and np.isnan(s[2]) and s[3] == 1


def test_more_rows_than_a_prompts_launch_can_count(built):
    hip = built.load()
    g = built.Gqa(16384, 1, 1, 16, 32, 16, 32, 2 ** 17, 1e-5, 0.1, 0.9, 8, 8, 8, 16, 16)
    with pytest.raises(built.BitNetHipError, match="too many for one launch"):
        hip.kv8_prefill_dev(g, 16, 16, 16, 16384 * 32, 2 ** 17, 2 ** 17, 16, 16384 * 32)
    assert hip.kv8_prefill_scratch_bytes(g, 2 ** 17, 2 ** 17) == 0
