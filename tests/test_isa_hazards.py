"""The wait states that gfx950 needs between dependent instructions, in every
kernel of the library (CPU only: the assembly of the objects built here)."""
import pytest

from rdnattention import _build
from tests import isa_hazards

pytestmark = pytest.mark.skipif(not all((isa_hazards.LLVM / t).exists() for t in
                                        ("llvm-objcopy", "llvm-objdump", "clang-offload-bundler")),
                                reason="needs ROCm's LLVM tools")

SOURCES = sorted(p.name for p in _build.CSRC.glob("*.hip"))


@pytest.fixture(scope="module")
def objects():
    if not all((_build.BUILD / "obj" / f"{s}.o").exists() for s in SOURCES):
        _build.build()
    return _build.BUILD / "obj"


@pytest.mark.parametrize("source", SOURCES)
def test_wait_states(objects, tmp_path, source):
    asm = isa_hazards.disassemble(objects / f"{source}.o", tmp_path)
    code = isa_hazards.kernels(asm)
    found = isa_hazards.report(code)
    assert not found, f"{len(found)} pairs too close, the first: " + "\n".join(found[:5])
    if "global_load_lds" in asm or "offen lds" in asm:  # the copies were read as such
        assert any(i.lds_copy for k in code.values() for i in k)


def lines(*text):
    return "0000000000001000 <kernel>:\n" + "".join(
        f"\t{t:<50} // {0x1000 + 4 * n:012X}: 00000000{tail}\n" for n, (t, tail) in
        enumerate((t if isinstance(t, tuple) else (t, "")) for t in text))


LOAD = "global_load_lds_dwordx4 v4, s[12:13]"


@pytest.mark.parametrize("want,code", [
    (0, ["s_mov_b32 m0, s3", "s_nop 0", LOAD]),
    (1, ["s_mov_b32 m0, s3", LOAD]),
    (1, ["v_readlane_b32 s13, v5, 0", "s_mov_b32 m0, s3", "s_nop 2", LOAD]),
    (0, ["v_readlane_b32 s13, v5, 0", "s_mov_b32 m0, s3", "s_nop 3", LOAD]),
    # copied by a scalar instruction: no longer the vector instruction's
    (0, ["v_readlane_b32 s5, v5, 0", "s_mov_b32 m0, s3", "s_mov_b64 s[12:13], s[4:5]", LOAD]),
    (0, ["v_readlane_b32 s13, v5, 0", "s_mov_b32 s13, 0", "s_mov_b32 m0, s3", "s_nop 0", LOAD]),
    # over a branch: the taken path is short, the other one is not
    (1, ["v_readfirstlane_b32 s12, v1", ("s_cbranch_scc1 4", " <kernel+0x18>"), "s_nop 4", "s_nop 4", "s_nop 4",
         "s_nop 4", "buffer_load_dword v1, s[12:15], 0 offen"]),
    # around a loop
    (1, ["buffer_load_dword v1, s[12:15], 0 offen", "s_nop 7", "v_readfirstlane_b32 s12, v1",
         ("s_cbranch_scc1 65532", " <kernel>"), "s_endpgm"]),
    (1, ["v_mfma_f32_32x32x16_f16 v[0:15], v[20:23], v[24:27], v[0:15]", "s_nop 7", "s_nop 2",
         "v_max3_f32 v30, v15, v31, v32"]),
    (0, ["v_mfma_f32_32x32x16_f16 v[0:15], v[20:23], v[24:27], v[0:15]", "s_nop 7", "s_nop 3",
         "v_max3_f32 v30, v15, v31, v32"]),
    (1, ["v_max3_f32 v30, v1, v2, v3", "s_nop 0", "v_permlane32_swap_b32_e32 v30, v31"]),
    (1, ["v_max3_f32 v30, v1, v2, v3", "v_mfma_f32_32x32x16_f16 v[0:15], v[28:31], v[24:27], v[0:15]"]),
])
def test_the_reading_of_the_assembly(want, code):
    assert len(isa_hazards.report(isa_hazards.kernels(lines(*code)))) == want
