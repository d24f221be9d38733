"""The assembly check's rule on registers that a vector-ALU instruction writes and a matrix instruction reads: two wait states for
each of its operands A, B and C, as the compiler keeps them for the matrix instructions it knows."""
import pytest

from hipkittens_amd import isa_check

ASM = """
_Z3fooPi:
	v_mov_b32_e32 {reg}, v99
{between}	v_mfma_f32_16x16x32_bf16 a[0:3], v[8:11], v[4:7], a[0:3]
"""


@pytest.mark.parametrize("reg", ["v8", "v11", "v4", "v7", "a2"])
@pytest.mark.parametrize("between,states", [("", 0), ("\ts_nop 0\n", 1), ("\tv_mov_b32_e32 v90, v91\n", 1), ("\ts_nop 1\n", 2)])
def test_operand_written_in_front(reg, between, states):
    asm = ASM.format(reg=reg, between=between)
    want = [] if states >= 2 else [(reg, states, 2)]
    assert [(f.register, f.wait_states, f.needed) for f in isa_check.scan(asm, sources=True)] == want
    assert [(f.register, f.wait_states, f.needed) for f in isa_check.check_texts({"foo": asm})] == want   # what the build asks for


def test_other_registers_do_not_count():
    assert isa_check.scan(ASM.format(reg="v12", between=""), sources=True) == []
