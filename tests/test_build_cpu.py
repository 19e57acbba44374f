"""The registers a thread that the compiler gave the kernels whose warps divide them among themselves (setmaxnreg): the shares are
written down for one number, and a kernel of another is not launched."""
import pytest

from yanlongvla_b200 import _lib, build

LOG = '''ptxas info    : 0 bytes gmem
ptxas info    : Compiling entry function '_Z13k_cross_tilesILi0ELi64ELb1EEvv' for 'sm_100a'
ptxas info    : Function properties for _Z13k_cross_tilesILi0ELi64ELb1EEvv
    8 bytes stack frame, 0 bytes spill stores, 0 bytes spill loads
ptxas info    : Used %d registers, used 16 barriers, 8 bytes cumulative stack size
ptxas info    : Compiling entry function '_Z16k_attention_manyILi0ELi64ELi1EEvv' for 'sm_100a'
ptxas info    : Used 128 registers, used 3 barriers
ptxas info    : Compiling entry function '_Z16k_attention_manyILi0ELi64ELi2EEvv' for 'sm_100a'
ptxas info    : Used %d registers, used 3 barriers
'''


def test_what_is_found_in_a_log():
    assert build.wrong_registers(LOG % (168, 80)) == []
    assert build.wrong_registers(LOG % (166, 80)) == [('_Z13k_cross_tilesILi0ELi64ELb1EEvv', 166, 168)]
    assert build.wrong_registers(LOG % (168, 72)) == [('_Z16k_attention_manyILi0ELi64ELi2EEvv', 72, 80)]


def test_the_numbers_are_those_of_the_sources():
    for name, want in (('cross_attention', 168), ('kv8_attention', 80)):
        text = (build.CSRC / f'{name}.cu').read_text()
        assert f'LAUNCH_REGS = {want}' in text and f'aligned.u32 {want};' in text
    assert sorted(build.LAUNCH_REGS.values()) == [80, 168]


@pytest.mark.parametrize('name,kernels', [('cross_attention', 24), ('kv8_attention', 12)])
def test_this_build(name, kernels):
    log = build.OBJ / f'{name}.ptxas'
    if not log.exists():
        pytest.skip('not built here')
    text = log.read_text()
    assert build.wrong_registers(text) == []
    assert len(build.registers(text)) == kernels                               # all of them were found


def test_the_status_says_so():
    assert b'registers' in _lib.lib.tcq_status_string(8) and _lib.lib.tcq_status_string(9) == b'unknown status'
