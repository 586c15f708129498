"""The sampler's CTAs write into each other's shared memory, which needs every
CTA of the cluster to have started: read off the kernel's source, as a run on a
GPU would show nothing but luck."""
import re
from pathlib import Path

SOURCE = (Path(__file__).resolve().parents[1] / "vllm_b200/csrc/tvp_sample.cu").read_text()


def body(name):
    """The text between the braces of function `name`, without comments."""
    text = re.sub(r"//[^\n]*", "", SOURCE)
    at = text.index("{", text.index(")", text.index(f" {name}(")))
    depth = 0
    for i in range(at, len(text)):
        depth += (text[i] == "{") - (text[i] == "}")
        if depth == 0:
            return text[at + 1:i]
    raise AssertionError(name)


def test_no_remote_access_before_every_cta_has_started():
    kernel = body("sample_kernel")
    remote = re.search(r"of_rank\(|map_shared_rank\(|share\(|::sync\(\)|Sampler<CL, RES> a\b", kernel)
    arrive = [m.start() for m in re.finditer(r"barrier_arrive\(\)", kernel)]
    wait = [m.start() for m in re.finditer(r"barrier_wait\(", kernel)]
    assert len(arrive) == len(wait) == 1
    assert arrive[0] < wait[0] < remote.start()
    # one arrival and one wait of every thread: no way around either of them
    before = kernel[:wait[0]]
    assert "return" not in before
    for at in (arrive[0], wait[0]):
        assert kernel[:at].count("{") == kernel[:at].count("}")
    # the arrival comes first, so that the wait hides behind the pass over the row
    assert "for (" not in kernel[:arrive[0]] and "__syncthreads" not in kernel[:arrive[0]]


def test_the_row_that_a_cluster_takes_is_found_without_remote_access():
    """It runs between the arrival and the wait."""
    assert not re.search(r"of_rank|map_shared_rank|this_cluster", body("in_turn"))
