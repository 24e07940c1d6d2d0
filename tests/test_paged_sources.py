"""What the paged kernels' sources must keep to where a run cannot show it: the failure paths of waits that never fail."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bonsai_pot_b200", "csrc")


def code(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_the_lanes_of_a_warp_decide_together_whether_a_wait_gave_up():
    """A lane that leaves a loop alone strands the others in its next shuffle. Outside of a vote a wait's result may only be dropped
    (every lane goes on), come before a barrier that all threads reach, or be looked at by one elected thread."""
    src = code("bp_kv4_attention.cu")
    waits = re.findall(r"[^\n]*\bwait_phase\([^\n]*", src)
    assert len(waits) >= 2
    for line in waits:
        assert "__all_sync(FULL, wait_phase(" in line or "(void)wait_phase(" in line, line
    src = code("bp_kv4_prefill.cu")
    expanders = src[src.index("const uint32_t quarter = lane >> 3, row"):src.index("const uint32_t x = (warp - S::FIRST_SOFTMAX)")]
    softmax = src[src.index("const uint32_t x = (warp - S::FIRST_SOFTMAX)"):src.index("done += n;")]
    for part, form in ((expanders, "__all_sync(FULL, waitx("), (softmax, "(void)waitx(")):
        waits = re.findall(r"[^\n]*\bwaitx\([^\n]*", part)
        assert len(waits) >= 2
        for line in waits:
            assert form in line, line


def test_who_makes_a_barrier_fences_it():
    """A fence orders the barriers that its own thread has made before the copies that arrive on them; another thread's does not."""
    src = code("bp_kv4_attention.cu")
    assert src.count("mbar_init(") == src.count("fence_barrier_init(") == 1
    assert re.search(r"if \(lane < RING\) \{\s*mbar_init\([^\n]*\);\s*fence_barrier_init\(\);\s*\}", src)
    src = code("bp_kv4_prefill.cu")
    blocks = re.findall(r"if \(threadIdx\.x == 0\) \{\n((?:    [^\n]*\n)+)  ?(?:  )?\}", src)
    made = [b for b in blocks if "mbar_init(" in b]
    assert len(made) == 2 and all("fence_barrier_init();" in b for b in made)
    assert sum(b.count("mbar_init(") for b in made) == src.count("mbar_init(")
