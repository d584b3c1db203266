"""CPU checks around the cache's attention: what the build verifies."""
from __future__ import annotations

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
