"""Attention over a paged cache against its definition in 64 bits.

Bound of an output value: half a step of bf16 (2^-8 of it) for the one rounding, and `soft` times sum_j p_j |v_j| for what the probabilities are off by, numerator and sum: twice the error of a
score (head_dim additions in 32 bits, 2^-24 of scale * sum |q_i k_i| each, and the score's own rounding times log2 e), and 2^-15 for the exponential, the probabilities' two bf16 parts and the
sums over the keys (added in 32 bits, a few thousand in a row at most before parts are joined)."""
import pytest
import torch

from hyperqwen_rtx4080s32_b200 import ops

pytestmark = pytest.mark.gpu


def bf16(*shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(torch.bfloat16)


def make(lens, news, hq, hk, d, rows, head_major=True, gated=False, seed=0, std=1.5):
    width = max([1] + [-(-n // rows) for n in lens])
    pages = sum(-(-n // rows) for n in lens) + 2
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).int()
    table, at = torch.full((len(lens), width), -5, dtype=torch.int32), 0        # what no key uses is not looked at
    for i, n in enumerate(lens):
        used = -(-n // rows)
        table[i, :used] = order[at:at + used]
        at += used
    cache = [bf16(pages, hk, rows, d, seed=seed + j).transpose(1, 2) if head_major else bf16(pages, rows, hk, d, seed=seed + j) for j in (1, 2)]
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    s = dict(q=bf16(starts[-1], hq, d, seed=seed + 3, std=std), k_pages=cache[0], v_pages=cache[1], page_table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    more = dict(q_starts=None if len(set(news)) == 1 else torch.tensor(starts, dtype=torch.int32, device="cuda"), gate=bf16(starts[-1], hq, 2 * d, seed=seed + 4)[..., d:] if gated else None)
    return s, more, starts


def want_and_bound(s, more, starts, scale=None):
    q, (hq, d) = s["q"].double(), s["q"].shape[1:]
    rows, hk = s["k_pages"].shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    want, slack = torch.zeros_like(q), torch.zeros_like(q)
    for b, n in enumerate(s["lens"].tolist()):
        new = starts[b + 1] - starts[b]
        if n <= 0 or new == 0:
            continue
        at = torch.arange(n, device="cuda")
        page = s["page_table"][b, at // rows].long()
        for h in range(hk):
            k, v = s["k_pages"][page, at % rows, h].double(), s["v_pages"][page, at % rows, h].double()
            g = slice(h * (hq // hk), (h + 1) * (hq // hk))
            for i in range(new):
                sees = n - new + i + 1
                if sees <= 0:
                    continue
                t = starts[b] + i
                score = scale * (q[t, g] @ k[:sees].T)
                size = (scale * (q[t, g].abs() @ k[:sees].abs().T)).amax(-1, keepdim=True)
                p = torch.softmax(score, -1)
                want[t, g] = p @ v[:sees]
                slack[t, g] = (2.0 ** -15 + 2 * (d + 8) * 2.0 ** -24 * size) * (p @ v[:sees].abs())
    if more.get("gate") is not None:
        gate = torch.sigmoid(more["gate"].double())
        want, slack = want * gate, slack * gate + 2.0 ** -20 * want.abs()
    return want, 2.0 ** -8 * want.abs() + slack


def check(got, s, more, starts, scale=None):
    want, bound = want_and_bound(s, more, starts, scale)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound.clamp_min(1e-30)).max()):.3g} of the bound"


CASES = [  # lens, new tokens, query heads, kv heads, head_dim, rows of a page
    ([1], [1], 1, 1, 64, 1), ([517], [1], 40, 8, 128, 16), ([64], [1], 8, 8, 64, 16), ([0, 1, 2], [1, 1, 1], 5, 1, 128, 16), ([15, 16, 17, 31, 33, 63, 64, 65, 127, 129], [1] * 10, 10, 2, 128, 16),
    ([300, 7, 0, 1000], [4] * 4, 24, 4, 256, 16), ([3, 2, 1, 4], [4] * 4, 6, 1, 256, 16), ([100, 5, 77, 400], [1, 3, 0, 5], 12, 3, 64, 24), ([4000], [1], 2, 1, 256, 64), ([9000, 30], [2, 2], 16, 2, 128, 48),
    ([257, 640], [1, 1], 17, 1, 128, 5), ([257, 640, 12], [2, 7, 12], 40, 8, 128, 16), ([700], [1], 64, 1, 128, 16), ([1200, 10], [33, 10], 6, 2, 64, 16), (list(range(0, 200, 3)), [1] * 67, 4, 4, 64, 8), ([20000], [1], 5, 1, 128, 16)]


@pytest.mark.parametrize("head_major", [True, False])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_the_definition(case, head_major):
    s, more, starts = make(*case, head_major=head_major, gated=case[4] == 256, seed=len(case[0]))
    got = ops.paged_attention(**s, **more)
    assert got.shape == s["q"].shape and got.is_contiguous()
    check(got, s, more, starts)
    assert torch.equal(got, ops.paged_attention(**s, **more))         # the same order of sums every time
    assert ops.device_status() == 0


def test_more_sequences_than_a_block_has_threads():
    lens = [(7 * i) % 41 for i in range(1300)]
    s, more, starts = make(lens, [1] * 1300, 2, 1, 64, 16)
    check(ops.paged_attention(**s, **more), s, more, starts)


@pytest.mark.parametrize("scale,std", [(1.0, 1.0), (0.01, 1.0), (30.0, 4.0)])
def test_scales_and_large_scores(scale, std):
    s, more, starts = make([333, 90], [1, 1], 10, 2, 128, 16, std=std)
    check(ops.paged_attention(**s, **more, scale=scale), s, more, starts, scale)


@pytest.mark.parametrize("d,news", [(128, [1, 1, 1]), (256, [4, 4, 4]), (64, [3, 3, 3])])
def test_what_is_masked_may_hold_anything(d, news):
    """Rows behind a sequence's last key, pages of others, keys that a later token of the same step sees and an earlier one does not."""
    s, more, starts = make([70, 33, 9], news, 6, 2, d, 16)
    clean = ops.paged_attention(**s, **more)
    for pages in (s["k_pages"], s["v_pages"]):
        used = torch.zeros(pages.shape[:2], dtype=torch.bool, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            at = torch.arange(n, device="cuda")
            used[s["page_table"][b, at // 16].long(), at % 16] = True
        for value in (float("nan"), float("inf"), -float("inf")):
            pages[~used] = value
            assert torch.equal(ops.paged_attention(**s, **more), clean)
    if news[0] > 1:
        for pages, value in ((s["v_pages"], float("inf")), (s["v_pages"], float("nan")), (s["k_pages"], float("nan"))):
            keep = pages.clone()
            for b, n in enumerate(s["lens"].tolist()):
                pages[int(s["page_table"][b, (n - 1) // 16]), (n - 1) % 16] = value
            got = ops.paged_attention(**s, **more)
            last = torch.tensor([x - 1 for x in starts[1:]])
            first = torch.ones(starts[-1], dtype=torch.bool)
            first[last] = False
            assert torch.equal(got[first.cuda()], clean[first.cuda()])
            assert not bool(got[last.cuda()].isfinite().any())
            pages.copy_(keep)
    assert ops.device_status() == 0


def test_a_visible_value_that_is_not_finite_reaches_the_rows_that_see_it():
    s, more, starts = make([40, 50], [1, 1], 4, 2, 64, 16)
    clean = ops.paged_attention(**s, **more)
    s["v_pages"][int(s["page_table"][0, 1]), 3, 1, 7] = float("inf")
    got = ops.paged_attention(**s, **more)
    assert torch.equal(got[1], clean[1]) and torch.equal(got[0, :2], clean[0, :2])
    assert not bool(got[0, 2:, 7].isfinite().any()) and bool(got[0, 2:, :7].isfinite().all())


def test_tokens_that_see_nothing_and_rows_that_belong_to_nobody():
    s, more, starts = make([0, 2, 5], [2, 3, 1], 4, 2, 128, 16)
    out = torch.full((9, 4, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    q = torch.cat([s["q"], bf16(3, 4, 128, seed=99)])
    got = ops.paged_attention(**dict(s, q=q), **more, out=out)
    assert got.data_ptr() == out.data_ptr() and bool((out[6:] == 3).all())
    assert bool((out[:3] == 0).all())                  # a sequence without keys, and a token in front of the first key
    check(out[:6], s, more, starts)
    assert bool((ops.paged_attention(**dict(s, q=q), **more)[6:] == 0).all())
    s["lens"] = torch.tensor([-3, 2, 5], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.paged_attention(**s, **more), out[:6])


def test_layouts_of_queries_gates_and_results():
    s, more, starts = make([90, 45], [2, 2], 12, 2, 128, 16, gated=True)
    want = ops.paged_attention(**s, **more)
    by_head = s["q"].transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.zeros(4, 12, 256, dtype=torch.bfloat16, device="cuda")
    wide[..., :128].copy_(s["q"])
    odd = torch.zeros(4, 12, 131, dtype=torch.bfloat16, device="cuda")
    odd[..., 3:].copy_(s["q"])
    for q in (by_head, wide[..., :128], odd[..., 3:]):
        assert torch.equal(ops.paged_attention(**dict(s, q=q), **more), want)
    gate = torch.zeros(12, 4, 133, dtype=torch.bfloat16, device="cuda")[..., 5:].transpose(0, 1)
    gate.copy_(more["gate"])
    out = torch.full((4, 12, 135), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention(**s, **dict(more, gate=gate), out=out[..., 1:129])
    assert torch.equal(out[..., 1:129], want) and bool((out[..., :1] == 9).all()) and bool((out[..., 129:] == 9).all())
    one = make([64], [1], 4, 4, 64, 16)
    check(ops.paged_attention(**dict(one[0], q=one[0]["q"].expand(1, 4, 64)), **one[1]), *one)


@pytest.mark.parametrize("bad", [-1, 1 << 30, "short"])
def test_a_page_outside_the_cache_and_a_length_beyond_the_table(bad):
    s, more, starts = make([100, 60, 20], [2, 2, 2], 6, 2, 128, 16)
    clean = ops.paged_attention(**s, **more)
    if bad == "short":
        s["lens"] = torch.tensor([113, 60, 20], dtype=torch.int32, device="cuda")
    else:
        s["page_table"][0, 3] = bad
    got = ops.paged_attention(**s, **more)
    first = 1 if bad == "short" else 0            # 7 pages hold 112 keys: the first of the two tokens sees no more than those
    assert bool(got[first:2].isnan().all()) and bool(got[:first].isfinite().all()) and torch.equal(got[2:], clean[2:])
    assert ops.device_status() == 2 and ops.device_status() == 0


def test_offsets_beyond_32_bits():
    rows, hk, d = 64, 8, 128
    pages = 40000                                   # 2.6e9 values in 5.2 GB, keys and values in the same pages
    cache = torch.zeros(pages, hk, rows, d, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    s, more, starts = make([200, 130], [1, 1], 16, hk, d, rows)
    old = s["k_pages"]
    where = torch.randperm(500)[:old.shape[0]].int().cuda()
    where = torch.where(where % 2 == 0, where, pages - 1 - where)
    cache[where.long()] = old
    table = s["page_table"].clone()
    used = table >= 0
    table[used] = where[table[used].long()]
    s = dict(s, k_pages=cache, v_pages=cache, page_table=table)
    check(ops.paged_attention(**s, **more), s, more, starts)


def test_captured_replayed_and_on_two_streams():
    a = make([700, 90], [1, 1], 10, 2, 128, 16, seed=1)
    b = make([300, 1500], [1, 1], 10, 2, 128, 16, seed=2)
    want = [ops.paged_attention(**x[0], **x[1]) for x in (a, b)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for st, x in zip(streams, (a, b)):
        st.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(ops.paged_attention(**x[0], **x[1]))
        graphs.append(g)
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    a[0]["lens"].copy_(torch.tensor([13, 90], dtype=torch.int32))            # the same graph, other lengths and queries
    a[0]["q"].copy_(bf16(2, 10, 128, seed=77))
    graphs[0].replay()
    torch.cuda.synchronize()
    check(outs[0], *a)
