"""Checks on the generated gfx950 code of csrc/dz_token_head.hip (no GPU needed).

Loads to LDS are written in assembly: they set M0, which the compiler is not told of, since M0 is a register that
a statement cannot reserve (naming it as overwritten is taken with a warning, and without a guarantee). That is
sound as long as the compiler keeps nothing of its own in M0, which these tests hold the generated code to: M0
is named by those statements alone, and no instruction that reads it without naming it stands outside of them.

Barriers that are written for a slab's loads wait for no reads of LDS: the places that are loaded next must have been
read before. Reads are waited for by the products that take them, which have to stand before the barrier.
"""
import os
import re
import subprocess

import pytest

from dizo_amd import build as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEAD = os.path.join(ROOT, "dizo_amd", "csrc", "dz_token_head.hip")
TO_LDS = [re.compile(r"s_mov_b32 m0, s\d+$"), re.compile(r"s_nop 0$"), re.compile(r"global_load_lds_dwordx4 ")]
# read M0 without naming it: loads to LDS, moves by index, messages, ordered and global data share, interpolation
READS_M0 = re.compile(r"(global|buffer|scratch)_load_lds_|buffer_load_\w+ .*\blds\b|[sv]_movrel|s_set_gpr_idx|s_sendmsg|ds_gws_|ds_ordered|ds_\w+_addtid|"
                      r"ds_(append|consume)|v_interp|.* gds\b")


@pytest.fixture(scope="module")
def asm(tmp_path_factory):
    try:
        cc = B.hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    out = tmp_path_factory.mktemp("asm") / "head.s"
    flags = [f for f in B.HIPCC_FLAGS if f not in ("-shared", "-fPIC")]
    subprocess.run([cc, *flags, "--cuda-device-only", "-S", HEAD, "-o", str(out)], check=True, capture_output=True, text=True)
    return out.read_text()


def statements(text):
    """{kernel: [(inline, [instructions]), ...]}: each statement in assembly by itself, what the compiler wrote in between as one."""
    kernels, cur = {}, None
    for raw in text.splitlines():
        if re.match(r"^_Z\S*:", raw):
            cur = kernels[raw.split(":")[0]] = [(False, [])]
        elif cur is None:
            continue
        elif raw.startswith(".Lfunc_end"):
            cur = None
        elif raw.strip().startswith(";;#ASMSTART"):
            cur.append((True, []))
        elif raw.strip().startswith(";;#ASMEND"):
            cur.append((False, []))
        else:
            s = raw.split(";")[0].strip()
            if s and not s.startswith(".") and not s.endswith(":"):
                cur[-1][1].append(s)
    return kernels


def m0_faults(kernels):
    out = []
    for name, parts in kernels.items():
        for inline, ins in parts:
            if inline and any("m0" in i or READS_M0.match(i) for i in ins):
                if len(ins) != 3 or not all(p.match(i) for p, i in zip(TO_LDS, ins)):
                    out.append((name, ins))
            elif not inline:
                out += [(name, i) for i in ins if re.search(r"\bm0\b", i) or READS_M0.match(i)]
    return out


def unread_at_barriers(kernels):
    """Barriers that the code comes to with reads of LDS not waited for, in the order of the code."""
    out = []
    for name, parts in kernels.items():
        pending = 0
        for _, ins in parts:
            for i in ins:
                if i.startswith("ds_read") or i.startswith("ds_load"):
                    pending += 1
                elif m := re.match(r"s_waitcnt .*lgkmcnt\((\d+)\)", i):
                    pending = min(pending, int(m[1]))
                elif i == "s_barrier" and pending:
                    out.append((name, pending))
    return out


def test_m0_is_used_by_the_loads_to_lds_alone(asm):
    kernels = statements(asm)
    loads = {n: sum(1 for inline, ins in p if inline and ins and ins[0].startswith("s_mov_b32 m0")) for n, p in kernels.items()}
    assert sum(loads.values()) > 100 and any(loads.values())
    assert not m0_faults(kernels), m0_faults(kernels)[:3]


def test_lds_is_read_before_it_is_loaded_again(asm):
    assert not unread_at_barriers(statements(asm)), unread_at_barriers(statements(asm))[:5]


def test_the_checks_find_what_they_look_for():
    good = "_Zk:\n;;#ASMSTART\n\ts_mov_b32 m0, s4\n\ts_nop 0\n\tglobal_load_lds_dwordx4 v1, s[2:3] nt\n;;#ASMEND\n\tds_read_b128 v[0:3], v4\n" \
           "\ts_waitcnt lgkmcnt(0)\n\ts_barrier\n.Lfunc_end0:\n"
    assert not m0_faults(statements(good)) and not unread_at_barriers(statements(good))
    for planted in ("\ts_mov_b32 m0, s1\n", "\tv_readlane_b32 s1, v1, m0\n", "\ts_sendmsg sendmsg(MSG_INTERRUPT)\n", "\tds_write_addtid_b32 v1\n",
                    "\tbuffer_load_dword v1, s[0:3], 0 offen lds\n", "\tv_movrels_b32_e32 v1, v2\n", "\tglobal_load_lds_dword v1, s[2:3]\n"):
        assert m0_faults(statements(good.replace("\ts_barrier\n", planted + "\ts_barrier\n"))), planted
    assert m0_faults(statements(good.replace("\ts_nop 0\n", "")))
    assert unread_at_barriers(statements(good.replace("lgkmcnt(0)", "lgkmcnt(1)"))) == [("_Zk", 1)]
