"""A CTA of a pair does not end while the other may still send an arrival to one of its barriers: read from the source, and the
waits' parities counted out."""
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parent.parent / "fastconv_b200" / "csrc" / "fc_ff_tc.cu").read_text()


def block_from(text, start):
    """The braced block that begins at or after `start`, and where it ends."""
    first = text.index("{", start)
    level = 0
    for i in range(first, len(text)):
        level += {"{": 1, "}": -1}.get(text[i], 0)
        if level == 0:
            return text[first:i + 1], i + 1
    raise AssertionError("unbalanced")


def after_the_tiles(role):
    """What a role (a warp's branch) does once its loop over tiles is over."""
    loop = role.index("for (uint32_t item = first;")
    return role[block_from(role, loop)[1]:]


def roles():
    kernel = block_from(SOURCE, SOURCE.index("ff_tc_kernel(const __grid_constant__"))[0]
    producer, end = block_from(kernel, kernel.index("if (warp == 0) {"))
    matrix, end = block_from(kernel, kernel.index("else if (warp == 1) {", end - 1))
    return producer, matrix


def test_every_barrier_that_the_other_cta_arrives_at_is_waited_for_in_the_end():
    producer, matrix = roles()
    ends = after_the_tiles(producer) + after_the_tiles(matrix)
    remote = set(re.findall(r"arrive_remote\(first_cta\((bar_\w+)\(", SOURCE))
    assert remote == {"bar_acc_empty", "bar_small_empty"}
    for name in remote | {"bar_empty"}:  # the ring's releases come from the matrix instructions of the first CTA
        assert re.search(rf"mbar_wait\({name}\(", ends), f"nobody waits for the last arrivals at {name}"


@pytest.mark.parametrize("uses", range(9))
def test_the_waits_of_two_further_uses_see_every_release(uses):
    """Two accumulators in turn: use c waits on barrier c & 1 for the phase ((c >> 1) & 1) ^ 1.  After `uses` uses the waits of two
    more stand until both barriers have had all their releases, and no longer."""
    total = [(uses + 1) // 2, uses // 2]

    def passes(done, c):  # parity p: the phase of that parity is over, i.e. the current phase is the other one
        return (done[c & 1] & 1) != (((c >> 1) & 1) ^ 1)

    for first in range(max(0, total[0] - 1), total[0] + 1):
        for second in range(max(0, total[1] - 1), total[1] + 1):
            through = passes([first, second], uses) and passes([first, second], uses + 1)
            assert through == ([first, second] == total)
