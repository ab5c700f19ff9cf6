"""Rules of the kernels' sources that no run shows."""
import os
import re

import pytest

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onyxia_b200", "csrc", "kernels")
ELECTING = [f for f in sorted(os.listdir(KERNELS)) if f.endswith(".cu") and "elect_one()" in open(os.path.join(KERNELS, f)).read()]


@pytest.mark.parametrize("name", ELECTING)
def test_all_lanes_come_to_an_election(name):
    """A bounded wait may run out for some lanes of a warp only. An election of one lane waits for all of them: nothing that a lane knows alone stands in front
    of it, and a loop with elections is not left by single lanes."""
    text = open(os.path.join(KERNELS, name)).read()
    assert not re.findall(r"&& elect_one\(\)", text)
    left = re.findall(r"if \(([^\n]*mbar_wait[^\n]*)\) \{\s*ok = false;\s*break;", text)
    assert all("__all_sync" in condition for condition in left), left


def test_products_of_a_tile_begin_behind_the_threads_of_all_its_halves():
    """Where two threads share a row, each scales some columns of the row's sums, and products add to all of them: the issuing warp waits for both before it issues either half's."""
    text = open(os.path.join(KERNELS, "differential_prefill.cu")).read()
    issues = text[text.index("else if (warp == kIssues)"):text.index("umma_weights(t_sum")]
    wait = issues.index("mbar_wait(w_full")
    loops = [m.start() for m in re.finditer(r"for \(int h = 0; h < kHalves; h\+\+\)", issues)]
    assert len(loops) == 2 and loops[0] < wait < loops[1]  # a loop of waits, then a loop of products


def test_values_behind_the_last_key_are_cleared_in_their_own_round():
    """A wait by parity is good for the round before it is over: where two places hold one tile's values, those before them are waited for first."""
    text = open(os.path.join(KERNELS, "differential_prefill.cu")).read()
    clears = text[text.index("may be no number"):text.index("st.shared.v4.b32")]
    assert 0 <= clears.find("kHalves == 2 && i > 0 && ok && !added(i - 1)") < clears.index("mbar_wait(v_full")
