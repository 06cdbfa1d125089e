"""A wait of the few-token 8-bit projection that gave up must not end its CTA over copies that are still on
their way: they would land in shared memory that is the sums', or another CTA's by then.

Every interleaving of the loads' issuer, their landing, the products' issuer and the end, with either wait
giving up at any moment, as a host model of the kernel's rule: whoever gave up, the CTA waits for each copy that
was sent before it goes on.  That the kernel keeps to it is read off the source
(megaattention_b200/csrc/linear_quant.cu); tests/test_linear_give_up_gpu.py lets a wait run out."""
import os
import re

import pytest

SRC = os.path.join(os.path.dirname(__file__), "..", "megaattention_b200", "csrc", "linear_quant.cu")


def _ends_over_copies(count, stages, all_wait):
    """The number of states in which the CTA goes on while a copy is outstanding.  ``all_wait``: what has been
    sent is waited for whichever role gave up, and not only by a producer that gave up itself."""
    start = (0, frozenset(), 0, "send", "take")              # sent, outstanding, taken, producer, issuer
    seen, todo, bad = {start}, [start], 0
    while todo:
        sent, out, taken, prod, iss = todo.pop()
        nxt = [(sent, out - {c}, taken, prod, iss) for c in out]                          # a copy lands
        if prod == "send":
            if sent == count:
                nxt.append((sent, out, taken, "over", iss))
            else:
                if sent < stages or taken > sent - stages:
                    nxt.append((sent + 1, out | {sent}, taken, prod, iss))
                else:
                    nxt.append((sent, out, taken, "gave up", iss))
        if iss == "take":
            if taken == count:
                nxt.append((sent, out, taken, prod, "over"))
            elif taken < sent and taken not in out:
                nxt.append((sent, out, taken + 1, prod, iss))
            else:
                nxt.append((sent, out, taken, prod, "gave up"))
        if prod != "send" and iss != "take":                                              # all meet behind the products
            waits = "gave up" in (prod, iss) if all_wait else prod == "gave up"
            bad += bool(out) and not waits
        for s in nxt:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return bad


@pytest.mark.parametrize("count,stages", [(1, 1), (1, 3), (3, 3), (3, 4), (5, 3), (7, 2)])
def test_no_copy_outlives_a_cta_that_gave_up(count, stages):
    assert _ends_over_copies(count, stages, all_wait=False) > 0      # the model sees what the rule is for
    assert _ends_over_copies(count, stages, all_wait=True) == 0


def test_the_kernel_keeps_to_the_rule():
    text = open(SRC).read()
    body = text[text.index("linear_narrow_kernel(const"):text.index("allow_smem(K kernel")]
    waits = re.findall(r"wait_bounded\([^;]*?(0x1\d)\)", body)
    assert sorted(waits) == ["0x10", "0x12", "0x13"]
    for site in waits:                                               # each of them is known to all
        assert re.search(r"!wait_bounded\([^;]*%s\)\) (\{ )?s_gave_up = 1;" % site, body), site
    assert re.search(r"s_sent = static_cast<uint32_t>\(sent\);", body[:body.index("0x12")])
    # they meet, then whoever gave up each stage's last copy is waited for, and they meet again
    assert re.search(r"0x13.*?__syncthreads\(\);\s+if \(s_gave_up\) \{[^}]*?if \(tid == 0\) wait_for_copies\(full, STAGES, "
                     r"static_cast<int>\(s_sent % STAGES\), s_sent / STAGES & 1u, 0x11\);\s+__syncthreads\(\);\s+\}",
                     body, flags=re.S)


@pytest.mark.parametrize("stages", [1, 2, 4, 5, 11])
def test_the_last_copy_into_each_stage_is_the_one_waited_for(stages):
    """wait_for_copies' parities: of stage i the lap of its last copy, and for a stage without one the parity that
    reads as over on a fresh barrier."""
    for sent in range(5 * stages):
        turn, parity = sent % stages, sent // stages & 1
        for i in range(stages):
            laps = [c // stages for c in range(sent) if c % stages == i]
            assert (parity if i < turn else parity ^ 1) == (laps[-1] & 1 if laps else 1)
