"""Values and calls at the edge of what the operators beside the layers take: infinities, gates that hold NaN, caches of nothing."""
import pytest
import torch

from hyperqwen_rtx4080s32_b200 import ops

import test_gpu_adapters as adapters
import test_gpu_heads as heads
import test_gpu_paged as paged

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("m,rank,bank", [(1, 8, 1), (5, 16, 3), (30, 64, 6), (150, 16, 2), (150, 128, 5)])
def test_inner_values_beyond_bf16_are_not_made_nan(m, rank, bank):
    """Row 0: an infinite activation against positive weights.  Last row: inner values of 3.4e38, which 32 bits hold and bf16 alone does not, against columns
    small enough for the result.  Both against the definition: signed infinities, and a value within the usual bound."""
    s = adapters.make(m, 256, (48, 37), rank, bank, seed=m)
    s["ids"][0] = s["ids"][m - 1] = bank - 1
    s["scales"].fill_(1.0)
    a, b = s["a"][bank - 1], s["b"][bank - 1]
    a.copy_(a.abs() + 2.0 ** -6)
    b[:20] = b[:20].abs() + 2.0 ** -6             # columns that become +inf, -inf, and (mixed signs) NaN
    b[20:40] = -b[20:40].abs() - 2.0 ** -6
    b[40:44, 0], b[40:44, 1:] = 1.0, -1.0
    s["x"][0, 77] = INF
    got = adapters.call(s)
    assert bool((got[0, :20] == INF).all()) and bool((got[0, 20:40] == -INF).all()) and bool(got[0, 40:44].isnan().all())
    s["x"][0, 77] = -INF
    got = adapters.call(s)
    assert bool((got[0, :20] == -INF).all()) and bool((got[0, 20:40] == INF).all())
    if m > 1:
        rest = torch.arange(1, m, device="cuda")
        s["x"][0, 77] = 0
        want, bound = adapters.want_and_bound(s)
        assert bool(((got.double() - want).abs() <= bound)[rest].all())
    # inner values between bf16's largest (0x1.fep127) and 32 bits': products of 0x1.fcp127 and 0x1.8p120, a sum that 32 bits hold exactly
    row = m - 1
    s["x"][row].zero_()
    s["x"][row, 3], s["x"][row, 200] = 2.0 ** 127, 2.0 ** 120
    a.zero_()
    a[:, 3], a[:, 200] = 1.984375, 1.5
    b.mul_(2.0 ** -110)
    b[40:44] = 0
    got = adapters.call(s)
    assert bool(got[row].isfinite().all())
    want, bound = adapters.want_and_bound(s)
    assert bool(((got.double() - want).abs() <= bound)[row].all()) and float(want[row].abs().max()) > 0


@pytest.mark.parametrize("d", [64, 72])
def test_a_cache_of_no_pages(d):
    s, how = heads.make(5, 4, 2, d, 24 if d == 72 else 32, seed=2)
    want = ops.qk_norm_rope(**s, **how)[0]
    none = torch.zeros(0, 16, 2, d, dtype=torch.bfloat16, device="cuda")
    slots = torch.full((5,), -1, device="cuda")
    assert torch.equal(ops.qk_norm_rope_store(**s, k_pages=none, v_pages=none.clone(), slots=slots, **how), want) and ops.device_status() == 0
    slots[2] = 0
    assert torch.equal(ops.qk_norm_rope_store(**s, k_pages=none, v_pages=none.clone(), slots=slots, **how), want)
    assert ops.device_status() == 2 and ops.device_status() == 0


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("value", [float("nan"), INF, -INF])
def test_a_gate_of_a_token_that_sees_nothing(d, value):
    """Tokens in front of the first key share a tile with tokens that see one, stand in tiles without a key, or in sequences without any."""
    lens, news = [1, 0, 2, 40, 300], [2, 3, 60, 42, 1]
    s, more, starts = paged.make(lens, news, 6, 2, d, 16, gated=True, seed=d)
    clean = ops.paged_attention(**s, **more)
    blind = torch.cat([torch.arange(n) < n - length for length, n in zip(lens, news)]).cuda()
    assert int(blind.sum()) == 64
    more["gate"][blind] = value
    got = ops.paged_attention(**s, **more)
    assert bool((got[blind] == 0).all()) and torch.equal(got, clean)
