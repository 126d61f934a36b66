"""tools/isa_check.py on made-up loops: what it lets pass and what it must not."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def tool():
    spec = importlib.util.spec_from_file_location("isa_check", os.path.join(ROOT, "tools", "isa_check.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


DMA, READ = ("global_load_lds_dwordx4", "v1, s[2:3]"), ("ds_read_b128", "v[0:3], v4")
WAIT, BARRIER = ("s_waitcnt", "vmcnt(0) lgkmcnt(0)"), ("s_barrier", "")


def program(*loops):
    """each loop: its instructions, then a branch back to the first of them (4 bytes each)"""
    out = []
    for body in loops:
        for m, o in body:
            out.append((4 * len(out), m, o, 0))
        out.append((4 * len(out), "s_cbranch_scc1", "", (-(len(body) + 1)) & 0xFFFF))
    return out


def found(tool, name, *loops):
    findings = []
    tool.check_function(name, program(*loops), findings)
    return findings


SHARED, PRIVATE, HOISTED = [WAIT, BARRIER, DMA, READ], [WAIT, DMA, READ], [DMA, READ]


def test_a_loop_of_shared_tiles_needs_wait_and_barrier(tool):
    assert not found(tool, "some_kernel", SHARED)
    assert found(tool, "some_kernel", PRIVATE) and found(tool, "some_kernel", HOISTED)
    assert found(tool, "some_kernel", [BARRIER, WAIT, DMA, READ])


@pytest.mark.parametrize("name", ["_ZN3fs216xattn_few_kernelINS_4XB16ELi64EEEv", "_ZN3fs217xattn_mass_kernelINS_4XB16ELi64EEEv"])
def test_private_tiles_need_the_wait(tool, name):
    assert not found(tool, name, PRIVATE)
    assert found(tool, name, HOISTED)


def test_the_backward_cannot_lose_the_barrier_of_its_shared_tiles(tool):
    name = "_ZN3fs216xattn_bwd_kernelINS_4XB16ELi128ELb0EEEvNS_5XArgsE"
    assert not found(tool, name, SHARED, PRIVATE) and not found(tool, name, PRIVATE, SHARED)
    assert found(tool, name, PRIVATE, PRIVATE)                # the barrier gone
    assert found(tool, name, HOISTED, PRIVATE)                # the wait hoisted out of the shared loop
    assert found(tool, name, SHARED, HOISTED)                 # ... out of a private one
    assert not found(tool, "_ZN3fs216xattn_bwd_kernelINS_4XF32ELi128ELb0EEEvNS_5XArgsE", [READ])          # fp32: no DMA


def test_counted_waits_allow_no_scratch(tool):
    assert any(k in "_ZN3fs217xattn_mass_kernelINS_4XB16ELi128ELi4EEEvNS_5XArgsE" for k in tool.NO_SCRATCH)
