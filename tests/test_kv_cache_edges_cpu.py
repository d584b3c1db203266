"""CPU checks around the cache's attention: what the build verifies, the division by
an invariant."""
from __future__ import annotations

import random

import pytest


def _log(used, dim=128, rows=8, groups=1):
    name = (f"_ZN3fa83dec13decode_kernelINS0_3CfgILi{dim}ELi2ELi{rows}ELi{groups}EEELb1EEEv14CUtensorMap"
            "_stS4_NS0_4ArgsE")
    return (f"ptxas info    : Compiling entry function '{name}' for 'sm_100a'\n"
            f"ptxas info    : Function properties for {name}\n"
            "    0 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads\n"
            f"ptxas info    : Used {used} registers, used 8 barriers\n")


def test_build_checks_the_register_split():
    from ada_cute_fp8_flash_attention_b200 import _build
    # 65536 / (blocks * threads): 2 x 256, 3 x 256, 2 x 384, 1 x 640
    good = _log(128) + _log(80, dim=64) + _log(80, rows=16, groups=2) + _log(96, rows=16, groups=4)
    assert _build.check_decode_registers(good) == 4
    assert _build.check_decode_registers("ptxas info    : Used 40 registers") == 0
    for bad in (_log(126), good + _log(72, rows=16, groups=2), _log(88, dim=64)):
        with pytest.raises(RuntimeError, match="registers a thread"):
            _build.check_decode_registers(bad)


def test_division_by_one_multiplication():
    """The formula of fa8_kv.cuh's Divisor, over the whole range that it is used in."""
    rng = random.Random(1)
    for d in [*range(1, 200), 1023, 1024, 1025, 65535, 1 << 20, (1 << 30) + 7, (1 << 31) - 1]:
        shift = (d - 1).bit_length()
        mul = (((1 << shift) - d) << 32) // d + 1
        assert mul < 1 << 32
        last = (1 << 31) - 1
        for x in [0, 1, d - 1, d, d + 1, 2 * d - 1, last, (last + 1) // d * d - 1,
                  *(rng.randrange(1 << 31) for _ in range(50))]:
            if 0 <= x <= last:
                total = (mul * x >> 32) + x
                assert total < 1 << 32 and total >> shift == x // d
