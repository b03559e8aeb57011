"""The warps of the policy loss's ring leave its loop together or not at all: a warp that stays while another leaves would wait at the next
barrier for good.  What they decide by has to be the same for all of them, so it comes out of a barrier; a wait that runs out cannot be
brought about at a chosen place, so this is checked on the source."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bamboo_b200", "csrc")


def ring():
    with open(os.path.join(CSRC, "post_training.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    at = text.index("policy_ring_kernel(const T* logits")
    return text[at:text.index("constexpr int RESCALE_THREADS", at)]


def test_warps_leave_the_ring_by_the_answer_of_a_barrier():
    body = ring()
    shared = set(re.findall(r"\b(s_\w+)", " ".join(re.findall(r"__shared__[^;]*;", body))))
    # no flag that a warp sets for the others once a wait of its own ran out
    assert not [m for m in re.findall(r"if \(!alive\)\s*(\w+)\s*=", body) if m in shared]
    loop = body[body.index("for (int it = 0;; ++it)"):]
    breaks = re.findall(r"if \(([^;]*)\) break;", loop[:loop.index("if (!alive) {")])
    leaving = [c for c in breaks if "row < 0" in c]
    assert len(leaving) == 1 and "row_barrier_any" in leaving[0]
    assert all("sp.nvec" in c for c in breaks if c not in leaving)          # the others end a thread's chunks
