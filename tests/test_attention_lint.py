"""The attention units' direct-to-LDS loads are inline assembly: the wait states that the compiler
does not keep for those, in the gfx950 code that the build left.  CPU only."""
from concurrent.futures import ThreadPoolExecutor

import pytest
from test_direct_load_lint import _assembly, lint_hazards, needs_tools

UNITS = tuple(f"attention_{kind}_{dtype}.hip" for kind in ("rows", "grad")
              for dtype in ("f32", "f16", "bf16"))


@pytest.fixture(scope="module")
def assembly(tmp_path_factory):
    into = tmp_path_factory.mktemp("asm")
    with ThreadPoolExecutor(max_workers=len(UNITS)) as pool:
        return dict(zip(UNITS, pool.map(lambda u: _assembly(u, into)[0], UNITS)))


def test_lint_catches_an_address_that_a_vector_instruction_just_wrote():
    bad = """
_Z1kv:
  v_readfirstlane_b32 s4, v1
  v_readfirstlane_b32 s5, v2
  s_mov_b32 m0, s6
  s_nop 0
  global_load_lds_dwordx4 v3, s[4:5]
"""
    assert len(lint_hazards(bad)[1]) == 2
    assert not lint_hazards(bad.replace("s_nop 0", "s_nop 3"))[1]


@needs_tools
def test_wait_states_ahead_of_loads_in_inline_assembly(assembly):
    for unit, text in assembly.items():
        loads, problems = lint_hazards(text)
        assert loads > 100, (unit, loads)
        assert not problems, f"{unit}:\n" + "\n".join(problems[:20])
