"""The forms that large and in-between calls of the operators beside the layers take, against the definitions in 64 bits: adapters where a block walks down several tiles
of rows, four tokens to a block of the head norms, chunks of prompts in attention, and every width of its tile at every head size.  Bounds are those of the files these tests borrow from."""
import pytest
import torch

from hyperqwen_rtx4080s32_b200 import ops

import test_gpu_adapters as adapters
import test_gpu_heads as heads
import test_gpu_paged as paged

pytestmark = pytest.mark.gpu


# ---- adapters: more tiles of 32 rows than walks (the blocks that the GPU holds over the 256-wide blocks of columns) ----

def id_patterns(m, bank):
    """One adapter; runs that end inside tiles of 16 and 32 and inside walks; every row another; none for long stretches."""
    runs, at = torch.empty(m, dtype=torch.int64), 0
    lengths = (1, 15, 32, 33, 7, 100, 64, 3, 200, 31)
    for i in range(m):
        if at >= m:
            break
        n = lengths[i % len(lengths)]
        runs[at:at + n] = i % (bank + 1) - 1
        at += n
    blocks = torch.arange(m) // 150 % (bank + 1) - 1
    return [torch.full((m,), bank - 1), runs, torch.arange(m) % bank, blocks]


WALKS = [(1100, 256, (9000,), 8, 3), (1100, 256, (8000, 1003), 24, 4), (1075, 512, (4001, 5000), 16, 2), (1100, 256, (6144, 2048, 2048), 64, 3), (1057, 256, (8200, 800), 128, 2), (2051, 256, (20000,), 16, 5)]


@pytest.mark.parametrize("shape", WALKS, ids=str)
def test_adapters_where_a_block_walks_down_the_rows(shape):
    m, k, n_outs, rank, bank = shape
    s = adapters.make(*shape, seed=rank)
    for ids in id_patterns(m, bank):
        s["ids"] = ids.cuda()
        got = adapters.call(s)
        adapters.check(got, s)
        y = s["base"].clone()
        assert torch.equal(adapters.call({**s, "base": y}, out=y), got)
        wide = torch.full((m, sum(n_outs) + 13), 5.0, dtype=torch.bfloat16, device="cuda")          # rows that start anywhere
        adapters.call(s, out=wide[:, 5:5 + sum(n_outs)])
        assert torch.equal(wide[:, 5:5 + sum(n_outs)], got) and bool((wide[:, :5] == 5).all()) and bool((wide[:, -8:] == 5).all())
    s["ids"][[0, 31, 500, m - 1]] = torch.tensor([bank, -2, 1 << 40, -5], device="cuda")
    bad = torch.zeros(m, dtype=torch.bool, device="cuda")
    bad[[0, 31, 500, m - 1]] = True
    broken = adapters.call(s)
    assert bool(broken[bad].isnan().all()) and torch.equal(broken[~bad], got[~bad])
    assert ops.device_status() == 2 and ops.device_status() == 0


# ---- norms and rotation from 2,048 tokens on ----

BATCHED = [(2048, 40, 8, 128, 128, False), (2049, 24, 4, 256, 64, True), (2050, 3, 2, 512, 512, False), (2051, 5, 3, 48, 16, True), (2051, 7, 2, 64, 0, False), (2050, 9, 4, 72, 24, True), (4097, 1, 1, 16, 16, False),
           (2049, 70, 3, 64, 16, False), (2051, 2, 2, 256, 250, True)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", BATCHED, ids=str)
def test_norm_and_rotation_of_many_tokens(case, interleaved):
    t, hq, hk, d, rot, gated = case
    for norm in (True, False):
        s, how = heads.make(t, hq, hk, d, rot, gated, norm=norm, seed=d + rot)
        (q, k), v = heads.want_of(s, how, interleaved)
        got = ops.qk_norm_rope(**s, **how, interleaved=interleaved)
        heads.near(got[0], q)
        heads.near(got[1], k)
        few = [torch.cat(x) for x in zip(*(ops.qk_norm_rope(**dict(s, qkv=s["qkv"][i:i + 1000], positions=s["positions"][i:i + 1000]), **how, interleaved=interleaved) for i in range(0, t, 1000)))]
        assert torch.equal(got[0], few[0]) and torch.equal(got[1], few[1])          # a token's result does not depend on how many there are
        # every place of a block without a slot, one of the last block beyond the cache, the others in any order
        rows, pages = 16, -(-t // 16) + 2
        k_pages, v_pages = heads.pages_of(pages, rows, hk, d, True, 5), heads.pages_of(pages, rows, hk, d, False, 6)
        before = [k_pages.clone(), v_pages.clone()]
        slots = torch.randperm(pages * rows, generator=torch.Generator().manual_seed(t))[:t]
        for i in (0, 5, 10, 15, 20, 21, 22, 23, 41, 42, t - 1):
            slots[i] = -1 - i
        slots[t - 2] = pages * rows + 3
        assert torch.equal(ops.qk_norm_rope_store(**s, k_pages=k_pages, v_pages=v_pages, slots=slots.cuda(), **how, interleaved=interleaved), got[0])
        there = ((slots >= 0) & (slots < pages * rows)).nonzero()[:, 0].cuda()
        page, row = slots.cuda()[there] // rows, slots.cuda()[there] % rows
        before[0][page, row], before[1][page, row] = got[1][there], v[there].to(torch.bfloat16)
        assert torch.equal(k_pages, before[0]) and torch.equal(v_pages, before[1])
        assert ops.device_status() == 2 and ops.device_status() == 0


# ---- attention ----

@pytest.mark.parametrize("rows", [16, 24, 5])
@pytest.mark.parametrize("group,new", [(6, 1), (6, 2), (5, 4), (6, 5), (20, 1), (6, 37)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_every_width_of_a_tile(d, group, new, rows):
    """Rows of a tile: 8, 16, 24 or 32, by a sequence's new tokens times the group; contexts that several blocks share, ones of a few keys, and none."""
    case = ([4000, 333, max(new - 2, 0), 64, new], [new] * 5, 2 * group, 2, d, rows)
    s, more, starts = paged.make(*case, gated=rows == 24, seed=d + new)
    got = ops.paged_attention(**s, **more)
    paged.check(got, s, more, starts)
    assert torch.equal(got, ops.paged_attention(**s, **more))
    news = [new, 0, new + 1, 1, max(new - 1, 0)]          # the same width for a ragged batch, where the average says so
    s, more, starts = paged.make(case[0], news, *case[2:], gated=rows == 24, seed=d + new)
    paged.check(ops.paged_attention(**s, **more), s, more, starts)
    assert ops.device_status() == 0


def chunk_bounds(s, more, starts):
    """paged.want_and_bound, all tokens of a sequence at once."""
    q, (hq, d) = s["q"].double(), s["q"].shape[1:]
    rows, hk = s["k_pages"].shape[1:3]
    want, slack, g = torch.zeros_like(q), torch.zeros_like(q), hq // hk
    for b, n in enumerate(s["lens"].tolist()):
        new = starts[b + 1] - starts[b]
        if n <= 0 or new == 0:
            continue
        at = torch.arange(n, device="cuda")
        hidden = at[None, :] > torch.arange(n - new, n, device="cuda")[:, None]
        page, tok = s["page_table"][b, at // rows].long(), slice(starts[b], starts[b + 1])
        for h in range(hk):
            k, v = s["k_pages"][page, at % rows, h].double(), s["v_pages"][page, at % rows, h].double()
            for head in range(h * g, (h + 1) * g):
                score = d ** -0.5 * (q[tok, head] @ k.T)
                size = (d ** -0.5 * (q[tok, head].abs() @ k.abs().T)).masked_fill(hidden, 0).amax(-1, keepdim=True)
                p = torch.softmax(score.masked_fill(hidden, -float("inf")), -1).nan_to_num(0)
                want[tok, head] = p @ v
                slack[tok, head] = (2.0 ** -15 + 2 * (d + 8) * 2.0 ** -24 * size) * (p @ v.abs())
    if more.get("gate") is not None:
        gate = torch.sigmoid(more["gate"].double())
        want, slack = want * gate, slack * gate + 2.0 ** -20 * want.abs()
    return want, 2.0 ** -8 * want.abs() + slack


CHUNKS = [([2500], [2500], 10, 2, 128, 16), ([3000], [600], 40, 8, 128, 16), ([700, 1300, 1, 40], [700, 600, 1, 3], 12, 2, 64, 24), ([1000, 1600], [640, 640], 12, 2, 256, 16), ([1500, 300, 20], [37, 20, 30], 24, 4, 256, 16),
          ([1024 + 50] + [10 + 37 * i for i in range(63)], [1024] + [1] * 63, 10, 2, 128, 16), ([2000] * 3, [700, 1, 0], 4, 4, 64, 16), ([900, 1500], [1000, 1500], 8, 1, 128, 32)]


@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: f"{len(c[0])}x{max(c[1])}of{max(c[0])}_{c[2]}_{c[3]}_{c[4]}")
def test_chunks_of_prompts(case):
    s, more, starts = paged.make(*case, gated=case[4] == 256, seed=7)
    got = ops.paged_attention(**s, **more)
    want, bound = chunk_bounds(s, more, starts)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound.clamp_min(1e-30)).max()):.3g} of the bound"
    assert torch.equal(got, ops.paged_attention(**s, **more)) and ops.device_status() == 0


def test_the_bounds_of_chunks_are_those_of_tokens():
    s, more, starts = paged.make([40, 3, 0, 9], [7, 5, 2, 9], 6, 2, 64, 16, gated=True, seed=3)
    for a, b in zip(chunk_bounds(s, more, starts), paged.want_and_bound(s, more, starts)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-300)
