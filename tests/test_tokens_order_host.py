"""What the kernels of a decoder's step may not do, seen in their source: read anything ahead of the wait for the launch before, or through the
non-coherent path, since every pointer that they are given may be what that launch writes."""
import os
import re

import pytest

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "thnets_b200", "csrc", "kernels")


def source(name):
    with open(os.path.join(KERNELS, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name,ahead", [("gemv_q4.cu", ("fetch();", "fetch_scales(tile0", ".load(")), ("rmsnorm.cu", ("stage(i,", "p.gain[c]", "load(base0")),
                                        ("kv_append.cu", ("p.pos[", "p.seq[")), ("paged_attn.cu", ("p.seq[", "positions(p,", "p.c.table + "))])
def test_nothing_is_read_ahead_of_the_wait(name, ahead):
    text = source(name)
    for body in re.split(r"__global__", text)[1:]:
        wait = body.index("pdl_enter();")
        for use in ahead:
            assert use not in body or body.index(use) > wait, (name, use)


@pytest.mark.parametrize("name", ["gemv_q4.cu", "rmsnorm.cu", "kv_append.cu", "paged_attn.cu"])
def test_nothing_is_read_through_the_non_coherent_path(name):
    assert not re.search(r"__ldg|ld\.global\.nc|__restrict__", source(name))
