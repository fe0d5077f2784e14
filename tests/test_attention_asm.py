"""Checks on the generated gfx950 code of csrc/dz_attention.hip (no GPU needed), for what the loads to LDS in assembly rest on:
see tests/test_head_asm.py, whose checks these are. A wave that takes keys for itself loads a place of its own again
without a barrier: its reads have to be waited for before the load, too."""
import os
import re
import subprocess

import pytest

from dizo_amd import build as B
from test_head_asm import m0_faults, statements, unread_at_barriers

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    try:
        cc = B.hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asm") / "attention.s"
    flags = [f for f in B.HIPCC_FLAGS if f not in ("-shared", "-fPIC")]
    subprocess.run([cc, *flags, "--cuda-device-only", "-S", os.path.join(ROOT, "dizo_amd", "csrc", "dz_attention.hip"), "-o", str(out)], check=True,
                   capture_output=True, text=True)
    return statements(out.read_text())


def test_m0_is_used_by_the_loads_to_lds_alone(kernels):
    assert sum(1 for p in kernels.values() for inline, ins in p if inline and ins and ins[0].startswith("s_mov_b32 m0")) > 100
    assert not m0_faults(kernels), m0_faults(kernels)[:3]


def test_lds_is_read_before_it_is_loaded_again(kernels):
    assert not unread_at_barriers(kernels), unread_at_barriers(kernels)[:5]


def unread_at_loads(kernels):
    """Loads to LDS that follow a read of LDS, of this wave's own code, that is not waited for, in kernels without a barrier between."""
    out = []
    for name, parts in kernels.items():
        if not re.search(r"attend_kernel\S+Lb1ELNS\S*5StoreE0E", name):  # by keys, operands: one place a wave
            continue
        pending = 0
        for inline, ins in parts:
            for i in ins:
                if re.match(r"ds_read_b(64_tr|128)", i):
                    pending += 1
                elif m := re.match(r"s_waitcnt .*lgkmcnt\((\d+)\)", i):
                    pending = min(pending, int(m[1]))
                elif inline and i.startswith("global_load_lds") and pending:
                    out.append((name, pending))
    return out


def test_a_waves_own_place_is_read_before_it_is_loaded_again(kernels):
    assert any(re.search(r"attend_kernel\S+Lb1ELNS\S*5StoreE0E", n) for n in kernels)
    assert not unread_at_loads(kernels), unread_at_loads(kernels)[:5]
