"""Vector instructions ahead of the execution mask that they need, in the assembly of the training kernels' own gfx950 code objects.

Where a block begins that lanes reach around a condition, the mask is widened again first.  The compiler has put copies of vector registers in front
of that when it was short of registers (seen: the row number of a lane, kept in an accumulator register for later; lanes that the condition had left out
stored to addresses made of what the register held before).  Only scalar instructions may stand there."""
import re

import pytest

from test_wait_states_cpu import _kernels
from turbodeberta_amd import _lib


def unmasked(code):
    """code: [(address, text, target of a branch or None)].  Vector instructions between a block's beginning, which s_cbranch_execz goes to, and the
    instruction there that widens the mask."""
    index = {address: i for i, (address, _, _) in enumerate(code)}
    bad = []
    for i in sorted({index[target] for _, text, target in code if text.startswith("s_cbranch_execz")}):
        seen = []
        for _, text, _ in code[i:]:
            if re.match(r"s_or_b64 exec, exec,", text):
                bad += seen
                break
            if text.startswith(("s_cbranch", "s_branch", "s_endpgm", "s_barrier")) or re.match(r"s_\w+ exec", text) or "saveexec" in text:
                break
            if text.startswith(("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")) and not text.startswith(("v_readlane", "v_writelane", "v_readfirstlane")):
                seen.append(text)
    return bad


def test_copies_stand_behind_the_mask(tmp_path):
    _lib.load()
    found, kernels = {}, 0
    for name, code in _kernels(tmp_path):
        if not re.search(r"tdb_train|norm_|dropout_", name):
            continue
        kernels += 1
        start = code[0][0]
        if bad := unmasked([(address - start, text, target) for address, text, target in code]):
            found[name] = bad
    assert kernels > 60
    assert not found, "\n".join(f"{n}: {b}" for n, b in found.items())


@pytest.mark.parametrize("first,found", [("v_accvgpr_write_b32 a1, v1", 1), ("s_mov_b32 s0, s1", 0)])
def test_a_copy_in_front_is_found(first, found):
    code = ["s_and_saveexec_b64 s[2:3], vcc", "s_cbranch_execz", "v_mov_b32 v1, v2", first, "s_mov_b32 s4, s5", "s_or_b64 exec, exec, s[2:3]", "v_mov_b32 v3, v4", "s_endpgm"]
    assert len(unmasked([(4 * i, text, 12 if "execz" in text else None) for i, text in enumerate(code)])) == found
