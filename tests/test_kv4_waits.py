"""The barrier waits of the attention kernels, by their source: a bounded wait can give up for one lane and not
for another, and the warp-wide instructions after it want all lanes, so each wait of a whole warp is voted on."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "webpytorch_b200", "csrc")


def _code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_waits_of_a_warp_are_voted_on():
    header = _code("kv4_attn.cuh")
    body = re.search(r"bool warp_wait\([^)]*\)\s*\{(.*?)\}", header, re.S).group(1)
    assert "__all_sync(0xffffffffu" in body and "mbar_wait" in body
    for name in ("kv4_attn.cu", "kv4_prompt.cu"):
        src = _code(name)
        assert src.count("warp_wait") >= 2
        # what is left of the plain waits: those that ignore the abort flag, after which no answer is used
        assert set(re.findall(r"mbar_\w*wait\w*", src)) <= {"mbar_wait_drain"}, name


def test_a_step_that_was_not_decoded_is_not_handed_on():
    src = _code("kv4_prompt.cu")
    arrive = src.index("mbar_arrive(kv ? v_full(st) : k_full(st))")
    assert re.search(r"if \(!ok\) break;\s*ptx::fence_async_smem\(\);\s*__syncwarp\(\);\s*if \(lane == 0\) ptx::$", src[:arrive])
