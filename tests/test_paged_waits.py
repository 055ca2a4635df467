"""CPU checks of the attention kernels' bounded waits, by their source: a wait
that runs out can't be brought about on a GPU without leaving work undone, so
the rules that keep it from becoming a hang are checked here.

* A warp whose lanes go on to votes or tensor memory instructions together
  gives a wait up together: every wait of such a role is one of the warp.
* A warp that gave up doesn't wait (or load) on: the result of a wait is used.
* Loads in flight land before the CTA ends, whoever gave up."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "edgeexpert_b200" / "csrc"


def code(name):
    return re.sub(r"//[^\n]*", "", (CSRC / name).read_text())


def roles():
    """The tensor kernel's loaders, MMA issue and row threads."""
    body = code("tf_prefix_tensor.cuh").split("void tensor_cta(", 1)[1]
    setup, rest = body.split("} else if (warp >= 5) {", 1)
    loaders, rest = rest.split("} else if (warp == 4) {", 1)
    issue, rows = rest.split("uint32_t mine = tmem", 1)
    return setup, loaders, issue, rows


def test_roles_of_whole_warps_give_up_together():
    setup, loaders, issue, rows = roles()
    assert re.search(r"wait_warp = .*__all_sync\(0xffffffffu, wait\(b, parity\)\)", setup)
    for role in (loaders, rows):
        assert "wait_warp(" in role
        assert not re.search(r"(?<!\w)wait\(", role)
    assert "if (elect_one()) {" in issue  # one thread alone: it may leave by itself


def test_no_wait_is_ignored():
    _, loaders, issue, rows = roles()
    for role in (loaders, issue, rows):
        for line in re.findall(r"[^\n;{}]*(?<!\w)(?:wait|wait_warp|o_ready)\([^\n]*", role):
            assert re.search(r"\b(ok|return|o_ready)\b.*=|return|ok &&", line), line
    stream = code("tf_prefix_stream.cuh").split("void stream_warp(", 1)[1]
    assert "__all_sync(0xffffffffu, mbar_wait_limited(" in stream
    for line in re.findall(r"[^\n]*\blanded\(\)[^\n]*\n[^\n]*", stream):
        assert re.search(r"ok = landed\(\);\s+if \(!ok\) break;", line), line


def test_the_tensor_loaders_see_their_loads_land():
    _, loaders, _, _ = roles()
    end = loaders.split("next_job(job, u);", 1)[1]
    assert re.search(r"issued = ok \? it : it - 1;\s*for .*issued - S::kSlots.*\s*mbar_wait_limited\(", end)


def test_a_streaming_warp_that_gave_up_lets_its_loads_land():
    stream = code("tf_prefix_stream.cuh").split("void stream_warp(", 1)[1]
    assert re.search(r"i < \(ok \? R - 1 : R\); \+\+i\) \{\s*mbar_wait_limited\(", stream)
