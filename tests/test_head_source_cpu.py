"""The order of the head's tensor-memory loads and their waits, read from the source: an
order that the compiler is free to change shows in no result until it does."""

import re

from conftest import ROOT

SOURCE = (ROOT / "macboost_b200" / "csrc" / "kernels_head.cu").read_text()


def _asm(text):
    """The asm statements of `text`, each up to its semicolon."""
    return re.findall(r"asm volatile\((.*?)\);\n", text, re.S)


def test_loads_from_tensor_memory_are_tied_to_their_wait():
    """A statement that loads from tensor memory either waits itself, or its registers are
    in-out operands of the statement that waits (tmem_issue and tmem_wait)."""
    body = {name: SOURCE[SOURCE.index(f"void {name}("):] for name in ("tmem_issue", "tmem_wait")}
    body = {name: text[:text.index("\n}\n") + 1] for name, text in body.items()}
    assert body["tmem_wait"].count('"+r"(r[') == 32
    alone = [a for a in _asm(SOURCE) if "tcgen05.ld" in a and "tcgen05.wait::ld" not in a]
    assert alone == _asm(body["tmem_issue"])
