"""Registers of the 8-bit KV cache's kernels (CPU: hipcc cross-compiles them to gfx950
assembly; no GPU needed): none spills a vector register, and each leaves its SIMD the waves
that its workgroups count on (512 registers of a lane shared by the waves of a SIMD)."""

import re

import pytest

from tests.test_codegen import _assembly, _registers, pytestmark  # noqa: F401


def _most(name):
    """The registers that a kernel may use."""
    d = re.match(r"_ZN2fp\d+k_paged8(?:_rows)?INS_\w+?ELi\dELi(\d+)E", name)
    if "k_paged8_rows" in name:
        return {64: 256, 128: 256, 256: 512}[int(d.group(1))]  # 2, 2 and 1 wave(s) per SIMD
    if "k_paged8_merge" in name:
        return 64  # 8
    if "k_paged8" in name:
        return {64: 168, 128: 256, 256: 256}[int(d.group(1))]  # 3, 2 and 2
    return 128  # the cache's rows: 4


@pytest.mark.parametrize("source,kernels", [("fp_paged8.hip", 92), ("fp_kvcache.hip", 37)])
def test_registers(source, kernels):
    checked = 0
    for name, (regs, spilled) in _registers(_assembly(source)).items():
        assert spilled == 0 and regs <= _most(name), (name, regs, spilled)
        checked += 1
    assert checked == kernels
