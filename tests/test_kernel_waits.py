"""What the sources of the kernels with bounded waits have to keep to, and no run of them shows."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sana_b200", "csrc")


def code(name):
    src = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", src, flags=re.S)


def test_a_barrier_object_is_initialised_once():
    """mbarrier.init on a live barrier object is undefined: the decaying attention goes through its barriers in one loop,
    which knows the arrivals of each."""
    assert len(re.findall(r"\bmbar_init\s*\(", code("la_decay_tc.cu"))) == 1
