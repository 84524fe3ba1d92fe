"""The build refuses a prompt kernel whose launch has fewer registers than its
warpgroups share out among themselves."""

import importlib.util
import os
import re

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "needle-rs_b200")


def _build():
    spec = importlib.util.spec_from_file_location("needle_build", os.path.join(PKG, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _log(*registers, name="_ZN2nd18kv4_prefill_kernelILi64ELi64E6__halfEEv"):
    return "".join(f"""ptxas info    : Compiling entry function '{name}' for 'sm_100a'
ptxas info    : Function properties for {name}
    32 bytes stack frame, 56 bytes spill stores, 88 bytes spill loads
ptxas info    : Used {n} registers, used 11 barriers, 18000 bytes smem
""" for n in registers)


def test_too_few_registers_end_the_build():
    b = _build()
    with open(os.path.join(PKG, "csrc", "kv4_prefill.cu")) as f:
        source = f.read()
    b.check_registers(source, _log(80, 80) + _log(40, name="_ZN2nd15kv4_join_kernelE"))
    b.check_registers(source, _log(77))  # allocated as 80
    for bad in (_log(72), _log(80, 72), _log(80, name="other"), ""):
        with pytest.raises(RuntimeError):
            b.check_registers(source, bad)


def test_the_shares_are_those_of_the_launch():
    with open(os.path.join(PKG, "csrc", "kv4_prefill.cu")) as f:
        source = f.read()
    n = {k: int(v) for k, v in re.findall(r"(PRE_REGS_[A-Z]+) = (\d+)", source)}
    assert 4 * n["PRE_REGS_ROWS"] + n["PRE_REGS_CODES"] + n["PRE_REGS_ISSUE"] <= 6 * n["PRE_REGS_LAUNCH"]
