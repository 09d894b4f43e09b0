"""The order of the block's kernels: what is launched behind the attention reads its finished result, where the parts' join has nothing to do as well."""
import pytest
import torch

from hyperqwen_rtx4080s32_b200 import ops

import test_gpu_block as blocks
import test_gpu_paged as paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[1], [64], [1, 17, 64, 40], list(range(1, 33)), [0, 0, 5]], ids=str)
def test_the_layer_behind_short_attention_reads_what_it_wrote(lens):
    """Sequences of up to 64 keys lie in one block each.  Captured with the layer behind it and replayed on a result that holds NaN."""
    att = blocks.block(False, hq=8, hk=2)
    s, more, _ = paged.make(lens, [1] * len(lens), 8, 2, 64, 16)
    buf = torch.empty(len(lens), 8, 64, dtype=torch.bfloat16, device="cuda")

    def step():
        return att.o(ops.paged_attention(**s, **more, out=buf).flatten(1))

    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph, stream=side):
        y = step()
    for turn in range(30):
        s["q"].copy_(paged.bf16(*s["q"].shape, seed=100 + turn))
        buf.fill_(float("nan"))
        y.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        one = ops.paged_attention(**s, **more)
        torch.cuda.synchronize()
        want = att.o(one.flatten(1))
        torch.cuda.synchronize()
        assert torch.equal(buf, one) and torch.equal(y, want)
    assert ops.device_status() == 0
