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


def test_a_cta_that_gives_up_waits_for_what_is_in_flight():
    """Copies into shared memory, and products that read it, end before a CTA leaves: the
    producer waits on every stage's barrier, the issuer of products on one of its own."""
    role = SOURCE[SOURCE.index("if (warp == 0) {"):SOURCE.index("if constexpr (F32) asm volatile(\"setmaxnreg.inc")]
    copies, products = role.split("} else if (warp == 1) {")
    call = re.search(r"wait\.settle\(full \+ 8 \* i, (.*?), t0\);", copies)
    assert call and call.group(1) == "i < s ? ph : ph ^ 1"
    assert re.search(r"if \(!ok\) \{[^}]*commit_here\(settled\);\s*wait\.settle\(settled, 0, ", products)


def test_parity_of_each_stages_last_copies():
    """The rule above against the barrier's definition: after `steps` steps over k stages,
    stage i is in phase (number of its steps); waiting for parity p returns when the phase
    before the present one has parity p, so it has to be that of the stage's last step --
    or, without a step, that of the phase before the first."""
    for k in range(1, 7):
        for steps in range(40):
            s, ph = steps % k, steps // k % 2
            for i in range(k):
                last = (steps - i + k - 1) // k - 1     # the stage's last step, -1: none
                assert (ph if i < s else ph ^ 1) == last % 2
