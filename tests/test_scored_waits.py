"""How the kernels behind the scores and the shared attention give up a wait, read from their text."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pulsar_b200", "csrc")


def _text(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_tensor_memory_is_freed_behind_the_work_in_flight():
    """A block that gave up a wait lets its copies and products land before it frees the tensor memory that they write."""
    for name in ("head_scores.cu", "attention_shared_tcgen05.cu"):
        order = re.findall(r"__nanosleep|tcgen05\.dealloc", _text(name))
        assert order[0] == "__nanosleep" and set(order[1:]) == {"tcgen05.dealloc"}, name


def test_no_wait_without_a_limit():
    """Barriers in memory are waited for through the bounded functions alone, and their answer is looked at."""
    for name in ("head_scores.cu", "attention_shared.cu", "attention_shared_tcgen05.cu"):
        text = _text(name)
        assert "mbarrier.try_wait" not in text and "mbarrier.test_wait" not in text and "mbar_try_wait" not in text, name
        assert not re.search(r"^\s*mbar_wait\w*\(", text, re.M), name
