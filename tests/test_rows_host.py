"""The row-wise operators as far as the host alone shows them: their sources, launches, modules.  No GPU needed."""
import glob
import os
import re

from compressgnn_amd import build


# ------------------------------------------------------------------------- sources --
def _assembly_blocks():
    """(file, text) of every asm statement's template among the sources, pieces joined."""
    for path in sorted(glob.glob(os.path.join(build.CSRC, "*"))):
        text = open(path).read()
        for found in re.finditer(r'\basm\s*(?:volatile\s*)?\(\s*((?:"(?:[^"\\]|\\.)*"\s*)+)', text):
            yield os.path.basename(path), "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', found[1]))


def test_wide_stores_in_assembly_keep_their_registers():
    """On gfx950 the data of a store of more than 8 bytes may not be written by the vector ALU within two wait states; the compiler does
    not see a store in assembly, so the two stand behind it in the same block (s_nop n gives n + 1)."""
    stores = 0
    for name, text in _assembly_blocks():
        steps = [step.strip() for step in re.split(r"\\n|;", text.replace("\\t", " ")) if step.strip()]
        for k, step in enumerate(steps):
            if re.match(r"(global|buffer|flat|scratch)_store_dwordx[34]\b", step):
                stores += 1
                waited = re.match(r"s_nop (\d+)$", steps[k + 1]) if k + 1 < len(steps) else None
                assert waited and int(waited[1]) + 1 >= 2, (name, text)
    assert stores
