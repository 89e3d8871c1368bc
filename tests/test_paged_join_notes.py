"""What the join of the paged attention relies on, read from the kernels' source: it follows the note of every worker and
the item that a note names, so both are written on every way through a main kernel, errors among them. (The ways that
end early need a fault to be taken, so no run shows them.)"""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "munet_b200", "csrc")


def kernels():
    found = {}
    for name in ("attention_paged.cu", "attention_paged_tile.cu"):
        text = open(os.path.join(CSRC, name)).read()
        text = re.sub(r"//[^\n]*", "", text)
        for m in re.finditer(r"__global__.*?(\w+_kernel)\(PagedArgs a\) \{", text, re.S):
            found[m.group(1)] = text[m.end():text.index("\n}\n", m.end())]
    return found


def test_all_main_kernels_are_looked_at():
    assert sorted(kernels()) == ["attention_paged_mma_kernel", "attention_paged_simt_kernel", "attention_paged_tile_kernel"]


@pytest.mark.parametrize("name", kernels())
def test_note_before_the_first_return(name):
    body = kernels()[name]
    returns = re.search(r"^(  |    )return;", body, re.M)  # of the kernel itself, not of a lambda in it
    note = re.search(r"a\.notes\[\w+(\.x)?\] = make_int2\(0, -1\)", body)
    assert note and note.start() < returns.start()


def test_the_leader_walks_on_when_a_wait_runs_out():
    """Its walk writes the items that the notes of other workers name."""
    loop = re.findall(r"while \((.*?walk\.next\(a, upto, g, s, true\).*?)\) \{", kernels()["attention_paged_tile_kernel"])
    assert loop == ["walk.next(a, upto, g, s, true)"]
    body = kernels()["attention_paged_tile_kernel"].split("while (walk.next(a, upto, g, s, true)) {")[1]
    body = body[:body.index("\n      }\n")]
    assert not re.search(r"^        (  )?break;", body, re.M)  # out of the walk's own loop
