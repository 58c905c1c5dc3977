"""The built library's matrix instructions and the wait states behind them (tools/isa_hazards.py --mfma): the compiler counts them over the blocks that lead to a
use and has missed a way through short conditional blocks."""
import importlib.util
import os
import shutil

import pytest

ROOT = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..")
spec = importlib.util.spec_from_file_location("isa_hazards", os.path.join(ROOT, "tools", "isa_hazards.py"))
hz = importlib.util.module_from_spec(spec)
spec.loader.exec_module(hz)

PRODUCT = "v_mfma_f32_16x16x32_bf16 v[38:41], v[26:29], v[62:65], v[30:33]"


def found(*lines):
    """addresses of 4 bytes a line, as the disassembler prints them"""
    text = "\n0000000000000000 <kernel>:\n" + "".join(f"\t{s:<60}// {4 * i:012X}: 00000000\n" for i, s in enumerate(lines))
    return [(w, use) for w, _, use in hz.scan_mfma(hz.parse_disassembly(text)["kernel"])]


def test_a_use_behind_a_branch_is_found():
    """the pattern that was compiled: the product ends one short block, its spill opens the block that both lead to"""
    other = ["v_mfma_f32_16x16x32_bf16 v[50:53], v[26:29], v[62:65], v[6:9]"] * 4 + ["s_nop 5"]
    store = "scratch_store_dwordx4 off, v[38:41], off offset:80"
    assert found(PRODUCT, f"s_cbranch_vccnz {len(other)}", *other, store, "s_endpgm") == [(1, store)]
    assert found(PRODUCT, "s_nop 7", f"s_cbranch_vccnz {len(other)}", *other, store, "s_endpgm") == []


def test_what_waits_and_what_does_not():
    read = "v_add_f32_e32 v1, v40, v2"
    assert found(PRODUCT, "s_nop 6", read, "s_endpgm") == [(7, read)]
    assert found(PRODUCT, "s_nop 7", read, "s_endpgm") == []
    write = "v_mov_b64_e32 v[40:41], v[2:3]"
    assert found(PRODUCT, write, "s_endpgm") == [(0, write)]
    operand = "v_mfma_f32_16x16x32_bf16 v[2:5], v[38:41], v[6:9], v[2:5]"
    assert found(PRODUCT, operand, "s_endpgm") == [(0, operand)]
    further = "v_mfma_f32_16x16x32_bf16 v[38:41], v[26:29], v[62:65], v[38:41]"
    assert found(PRODUCT, further, "s_nop 7", read, "s_endpgm") == []
    assert found(PRODUCT, "v_add_f32_e32 v1, v42, v2", "ds_read_b128 v[38:41], v1", "s_endpgm") == []
    back = [read, PRODUCT, "s_cbranch_scc0 65533", "s_endpgm"]   # a loop: the next turn's first instruction
    assert found(*back) == [(1, read)]


def test_no_early_use_in_the_library():
    import vms_hip
    if shutil.which(hz.OBJDUMP) is None:
        pytest.skip("no llvm-objdump")
    kernels = hz.disassembly(vms_hip.LIB_PATH)
    assert any("gd_grad_kernel" in n for n in kernels) and any("gd_scan_kernel" in n for n in kernels)
    bad = {n: r for n, body in kernels.items() if (r := hz.scan_mfma(body))}
    assert not bad, bad
