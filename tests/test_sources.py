"""Properties of the kernels' sources that no run shows."""
import re

from conftest import ROOT

CSRC = ROOT / "block-gqt-webgpu_amd" / "csrc"


def _asm_blocks(text):
    """The bodies of inline asm statements (between the outer parentheses)."""
    for m in re.finditer(r"\basm(?:\s+volatile)?\s*\(", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"(": 1, ")": -1}.get(text[at], 0)
            at += 1
        yield text[m.end():at - 1]


def test_loads_in_inline_asm_wait_for_themselves():
    """The compiler takes an asm statement's outputs as written when it ends, so a load that is still in flight there
    could land in a register that holds something else by then: such a statement ends with its own wait."""
    seen = 0
    for path in sorted([*CSRC.glob("*.h"), *CSRC.glob("*.hip")]):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for block in _asm_blocks(text):
            code = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', block)).replace(r"\n", " ").replace(r"\t", " ")
            loads = list(re.finditer(r"\b(ds_read|ds_load|buffer_load|global_load|flat_load|scratch_load|s_load|s_buffer_load)\w*", code))
            if not loads:
                continue
            seen += 1
            wait = code.rfind("s_waitcnt")
            assert wait > loads[-1].start(), f"{path.name}: {code[:80]}"
            counter = "lgkmcnt(0)" if loads[-1].group(1).startswith(("ds_", "s_")) else "vmcnt(0)"
            assert counter in code[wait:wait + 60], f"{path.name}: {code[wait:wait + 40]}"
    assert seen >= 2  # (the transposed LDS reads)
