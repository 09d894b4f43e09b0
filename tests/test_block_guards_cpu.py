"""Guards of the operators beside the layers that need no GPU: the order of programmatic launches, refusals, files and banks."""
import os
import re

import pytest
import torch

from hyperqwen_rtx4080s32_b200 import ops

import test_block_ops_cpu as refusals

E, h = ops.GqError, refusals.h
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hyperqwen-rtx4080s32_b200", "csrc")


def kernels(text):
    """(name, body) of every __global__ function with a body, comments left out."""
    text = re.sub(r"//[^\n]*", "", text)
    for m in re.finditer(r"__global__", text):
        at = text.index("{", m.end())
        name = re.search(r"(\w+)\s*\(", re.sub(r"__launch_bounds__\((?:[^()]|\([^()]*\))*\)", "", text[m.end():at])).group(1)
        depth, end = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield name, text[at:end]


@pytest.mark.parametrize("header", ["gq_adapters.cuh", "gq_heads.cuh", "gq_paged.cuh"])
def test_every_kernel_waits_for_the_one_in_front_on_every_path(header):
    """These kernels are launched programmatically, and some let the next one start at once.  A kernel that ends without the wait may end before the
    kernel in front of it does, and what is launched behind it waits for it alone: so the wait stands in front of the first return, and in no branch."""
    with open(os.path.join(CSRC, header), encoding="utf-8") as f:
        found = list(kernels(f.read()))
    assert found
    for name, body in found:
        assert body.count("pdl_wait();") == 1, name
        ahead = body[:body.index("pdl_wait();")]
        assert "return" not in ahead, f"{name} returns before it has waited"
        assert ahead.count("{") - ahead.count("}") == 1 and ahead.rstrip()[-1] in ";}", f"{name} waits in a branch"


@pytest.mark.parametrize("missing", [("k_pages",), ("v_pages",), ("slots",), ("k_pages", "slots"), ("k_pages", "v_pages", "slots")], ids=str)
def test_a_store_without_a_part_of_its_cache_is_refused(missing):
    with pytest.raises(E, match="all given"):
        refusals.heads(store=True, **{name: None for name in missing})
