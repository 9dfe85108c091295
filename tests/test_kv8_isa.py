"""Registers of the kernels over caches of 8 bits (CPU only: hipcc cross-compiles): what their launches count on, in exactly the instances that launches choose."""
import os

import pytest

from tests.test_isa_guard import HIPCC, _compile


def test_caches_of_eight_bits_fit_their_registers(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("no hipcc")
    _, usage = _compile("kernels_kv8.hip", str(tmp_path))

    def found(kernel, count):
        some = {name: u for name, u in usage.items() if kernel in name}
        assert len(some) == count, (kernel, len(some))
        return some.items()

    for name, u in found("k_kv8_prefill", 28):  # two waves per SIMD; one of heads above 128 columns, and where LDS holds one workgroup of four waves
        alone = "ILi4ELi16E" in name or "ILi2ELi8ELi2ELb0ELi1ELi4E" in name
        assert u["ScratchSize"] == 0 and u["Occupancy"] >= (1 if alone else 2) and u["VGPRs"] + u["AGPRs"] <= (488 if alone else 254), (name, u)
    for name, u in found("k_kv8_step", 8):
        held = 1 if "ILi4E" in name or "ILi2ELi8ELi2E" in name else 2  # (step_held)
        assert u["ScratchSize"] <= (64 if "ILi4ELi16ELi2E" in name else 0) and u["Occupancy"] >= held, (name, u)
    for name, u in found("k_kv8_rows", 56):
        assert u["ScratchSize"] == 0 and u["Occupancy"] >= 2, (name, u)
    for name, u in found("k_kv8_read", 2):
        assert u["ScratchSize"] == 0 and u["Occupancy"] >= 8, (name, u)
