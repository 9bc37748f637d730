"""CPU: the check of the generated ISA for scalars written by vector instructions too shortly in front of an LDS-DMA that reads them in an asm
statement (build.py), on small kernels written here."""
import pytest

from fitclip_amd import build

DMA = "\tglobal_load_lds_dwordx4 v1, s[4:5]"


def _audit(tmp_path, body, name="k"):
    asm = tmp_path / "kernel.s"
    asm.write_text(f"\t.globl\tother\nother:                                  ; @other\n\ts_endpgm\n.Lfunc_end0:\n"
                   f"{name}:                                      ; @{name}\n; %bb.0:\n{body}\n.Lfunc_end1:\n\t.size\t{name}, .Lfunc_end1-{name}\n")
    return build.audit_asm_dma_hazards(asm, ["k"])


@pytest.mark.parametrize("body,dmas", [
    (f"\ts_mov_b32 s4, s8\n{DMA}\n\ts_endpgm", 1),                                                      # interlocked
    (f"\tv_readlane_b32 s4, v9, 0\n\ts_nop 4\n{DMA}\n\ts_endpgm", 1),                                   # five wait states
    (f"\tv_readlane_b32 s4, v9, 0\n\ts_mov_b32 s4, s8\n{DMA}\n\ts_endpgm", 1) ,                         # written again by the scalar unit
    (f"\tv_readlane_b32 s6, v9, 0\n{DMA}\n\ts_endpgm", 1),                                              # another register
    (f"\tv_readlane_b32 s4, v9, 0\n\ts_branch .LBB0_2\n.LBB0_1:\n{DMA}\n\ts_endpgm\n.LBB0_2:\n\ts_nop 3\n\ts_branch .LBB0_1", 1),
    (f"\ts_cbranch_scc1 .LBB0_1\n\ts_endpgm\n.LBB0_1:\n{DMA}\n\ts_nop 0\n{DMA}\n\ts_endpgm", 2),        # behind the first end: counted
    (f"\tv_readlane_b32 s4, v9, 0\n\ts_endpgm\n.LBB0_1:\n{DMA}\n\ts_branch .LBB0_1", 1),                # an end is no way on
])
def test_what_passes(tmp_path, body, dmas):
    assert _audit(tmp_path, body) == dmas


@pytest.mark.parametrize("body", [
    f"\tv_readlane_b32 s4, v9, 0\n{DMA}\n\ts_endpgm",
    f"\tv_readlane_b32 s5, v9, 0\n\ts_nop 3\n{DMA}\n\ts_endpgm",                                                      # four wait states
    f"\ts_cbranch_scc1 .LBB0_1\n\ts_endpgm\n.LBB0_1:\n\tv_readfirstlane_b32 s4, v9\n\ts_nop 0\n{DMA}\n\ts_endpgm",    # behind the first end
    f"\tv_readlane_b32 s4, v9, 0\n\ts_cbranch_scc1 .LBB0_1\n\ts_endpgm\n.LBB0_1:\n{DMA}\n\ts_endpgm",                 # across a branch
    f".LBB0_1:\n{DMA}\n\tv_readlane_b32 s4, v9, 0\n\ts_cbranch_scc1 .LBB0_1\n\ts_endpgm",                             # round a loop
    f"\tv_readlane_b32 s4, v9, 0\n.LBB0_1:\n\ts_nop 1\n{DMA}\n\ts_mov_b32 s4, s8\n\ts_branch .LBB0_1",                # from one of two ways
    f"\tv_readlane_b32 s4, v9, 0\n\ts_cmp_lt_i32 s4, s5\n{DMA}\n\ts_endpgm",                                          # a comparison writes nothing
    f"\tv_add_co_u32_e64 v2, s[4:5], v3, v4\n{DMA}\n\ts_endpgm",                                                      # the carry
    f"\tv_cmp_lt_u32_e64 s[4:5], v3, v4\n{DMA}\n\ts_endpgm",
    "\tv_cmp_lt_u32_e32 vcc, v3, v4\n\tglobal_load_lds_dword v1, vcc\n\ts_endpgm",
    "\tv_readlane_b32 s7, v9, 0\n\tbuffer_load_dwordx4 v1, s[4:7], 0 offen lds\n\ts_endpgm",
])
def test_what_is_found(tmp_path, body):
    with pytest.raises(RuntimeError, match="writes an SGPR"):
        _audit(tmp_path, body)


@pytest.mark.parametrize("body", [f"\ts_setpc_b64 s[30:31]\n{DMA}\n\ts_endpgm", f"\ts_branch .LBB9_9\n{DMA}\n\ts_endpgm", "\ts_endpgm"])
def test_what_the_audit_does_not_know_is_an_error(tmp_path, body):
    with pytest.raises(RuntimeError, match="out of date"):
        _audit(tmp_path, body)


def test_every_instruction_of_the_built_kernels_is_looked_at():
    import re
    found = 0
    for src, kernels in build.ASM_DMA_AUDIT.items():
        asm = build.CSRC / "build" / f"{src.replace('.hip', '')}-hip-amdgcn-amd-amdhsa-{build.ARCH}.s"
        if asm.exists():  # (built here)
            found += 1
            assert build.audit_asm_dma_hazards(asm, kernels) == len(re.findall(r"^\s+(?:global_load_lds_dword.*|buffer_load_dword.* lds)\s*(?:;.*)?$", asm.read_text(), flags=re.M))
    if not found:
        pytest.skip("no generated ISA beside the sources")
