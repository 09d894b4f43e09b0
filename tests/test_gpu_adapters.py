"""Low-rank adapters beside a shared projection against their definition in 64 bits.

Bound of an output value: half a step of bf16 (2^-8 of it) for the one rounding; for the sums in 32 bits 2^-24 per addition of the absolute terms, K of them in the inner
products, the rank's in the outer ones, and a few for what parts are added; the inner values enter the outer products as two bf16 parts, 2^-16 of them off at most."""
import pytest
import torch

from hyperqwen_rtx4080s32_b200 import ops

pytestmark = pytest.mark.gpu


def bf16(*shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(torch.bfloat16)


def make(m, k, n_outs, rank, bank, seed=0):
    n, shards = sum(n_outs), len(n_outs)
    g = torch.Generator(device="cuda").manual_seed(seed + 90)
    return dict(x=bf16(m, k, seed=seed + 1), base=bf16(m, n, seed=seed + 2), a=bf16(bank, shards * rank, k, seed=seed + 3, std=k ** -0.5),
                b=bf16(bank, n, rank, seed=seed + 4, std=rank ** -0.5), scales=0.5 + torch.rand(bank, shards, device="cuda", generator=g),
                ids=torch.randint(-1, bank, (m,), device="cuda", generator=g), n_outs=list(n_outs))


def want_and_bound(s, ids=None):
    ids = (s["ids"] if ids is None else ids).tolist()
    want, slack = s["base"].double(), s["base"].double().abs()
    rank, k = s["b"].shape[2], s["x"].shape[1]
    soft = torch.zeros_like(want)
    for m, i in enumerate(ids):
        if i < 0:
            continue
        at = 0
        for j, n in enumerate(s["n_outs"]):
            a, b, scale = s["a"][i, j * rank:(j + 1) * rank].double(), s["b"][i, at:at + n].double(), float(s["scales"][i, j])
            x = s["x"][m].double()
            inner = a @ x
            want[m, at:at + n] += scale * (b @ inner)
            slack[m, at:at + n] += scale * (b.abs() @ (a.abs() @ x.abs()))
            soft[m, at:at + n] += scale * (b.abs() @ inner.abs())
            at += n
    return want, 2.0 ** -8 * want.abs() + (k + rank + 16) * 2.0 ** -24 * slack + 2.0 ** -15 * soft


def call(s, **more):
    return ops.low_rank_add(s["base"], s["x"], s["a"], s["b"], s["scales"], s["ids"], s["n_outs"], **more)


def check(got, s, ids=None):
    want, bound = want_and_bound(s, ids)
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), f"worst {float((err / bound.clamp_min(1e-30)).max()):.3g} of the bound"


SHAPES = [(1, 256, (8,), 8, 1), (1, 5120, (5120, 1024, 1024), 16, 4), (2, 512, (1,), 16, 2), (5, 512, (96, 70, 64), 16, 3), (8, 256, (0, 40, 24), 32, 2), (17, 768, (33, 31), 8, 9),
          (27, 5120, (2176, 2176), 32, 8), (33, 1280, (333,), 24, 4), (64, 4352, (640,), 64, 16), (65, 512, (320,), 40, 3), (130, 768, (257, 255), 128, 2), (300, 512, (1000, 40, 8, 8), 56, 7),
          (1037, 1024, (512, 264), 16, 5), (70, 256, (64,) * 8, 128, 3)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_definition(shape):
    s = make(*shape)
    check(call(s), s)
    s["ids"] = s["ids"].int()
    first = call(s)
    check(first, s)
    assert torch.equal(first, call(s))              # the same order of sums every time
    assert ops.device_status() == 0


@pytest.mark.parametrize("m", [1, 9, 40, 200])
def test_ids_in_any_pattern(m):
    s = make(m, 512, (200, 56), 16, 6, seed=m)
    for ids in (torch.full((m,), -1), torch.full((m,), 5), torch.arange(m) % 6, torch.arange(m) // max(1, m // 3) % 6, torch.arange(m) % 7 - 1):
        s["ids"] = ids.cuda()
        check(call(s), s)
    s["ids"] = torch.full((m,), -1, device="cuda")
    assert torch.equal(call(s), s["base"])


def test_in_place_and_in_columns_of_a_wider_buffer():
    s = make(21, 512, (96, 71), 16, 4)
    want = call(s)
    for at in (0, 3, 8):
        wide = torch.full((21, 190), 7.0, dtype=torch.bfloat16, device="cuda")
        view = wide[:, at:at + 167]
        call(s, out=view)
        assert torch.equal(view, want)
        view.copy_(s["base"])
        assert ops.low_rank_add(view, s["x"], s["a"], s["b"], s["scales"], s["ids"], s["n_outs"], out=view).data_ptr() == view.data_ptr()
        assert torch.equal(view, want)
        assert bool((wide[:, :at] == 7).all()) and bool((wide[:, at + 167:] == 7).all())
    beside = torch.empty(21, 2 * 167, dtype=torch.bfloat16, device="cuda")       # base and out as columns of one buffer
    beside[:, :167].copy_(s["base"])
    assert torch.equal(ops.low_rank_add(beside[:, :167], s["x"], s["a"], s["b"], s["scales"], s["ids"], s["n_outs"], out=beside[:, 167:]), want)
    odd = torch.empty(21, 520, dtype=torch.bfloat16, device="cuda")[:, 5:517]    # inputs that start anywhere, and rows of one
    odd.copy_(s["x"])
    assert torch.equal(call(dict(s, x=odd)), want)
    s["x"], s["ids"] = s["x"][:1].expand(21, 512), s["ids"][:1].expand(21)
    check(call(s), s)


@pytest.mark.parametrize("m", [3, 50, 150])
def test_an_id_outside_the_bank_and_what_other_rows_see_of_it(m):
    s = make(m, 256, (64, 30), 16, 3, seed=7)
    good = call(s)
    bad = s["ids"].clone()
    bad[1], bad[m - 1] = 3, -2
    assert ops.device_status() == 0
    got = call(dict(s, ids=bad))
    assert bool(got[1].isnan().all()) and bool(got[m - 1].isnan().all())
    keep = torch.ones(m, dtype=torch.bool)
    keep[1] = keep[m - 1] = False
    want, bound = want_and_bound(s)
    assert bool(((got.double() - want).abs() <= bound)[keep.cuda()].all())
    assert ops.device_status() == 2 and ops.device_status() == 0
    assert good.isfinite().all()


@pytest.mark.parametrize("m", [6, 40, 150])
def test_weights_that_are_not_finite_reach_their_own_rows_only(m):
    s = make(m, 256, (64, 64), 16, 4, seed=3)
    s["ids"] = torch.arange(m, device="cuda") % 4
    s["a"][2] = float("nan")
    s["b"][2] = float("inf")
    s["x"][0, 5] = float("inf")                  # row 0 has adapter 0
    got = call(s)
    mine = (s["ids"] == 2)
    assert bool(got[mine].isnan().all()) and bool((~got[0].isfinite()).all())
    rest = ~mine
    rest[0] = False
    s["a"][2], s["b"][2], s["x"][0, 5] = 0, 0, 0
    want, bound = want_and_bound(s)
    assert bool(((got.double() - want).abs() <= bound)[rest].all())


def test_offsets_beyond_32_bits():
    k, rank, bank, n = 17408, 128, 1000, 64
    a = torch.zeros(bank, rank, k, dtype=torch.bfloat16, device="cuda")       # 2.2e9 values
    s = make(3, k, (n,), rank, 1, seed=11)
    a[bank - 1] = s["a"][0]
    b = torch.zeros(bank, n, rank, dtype=torch.bfloat16, device="cuda")
    b[bank - 1] = s["b"][0]
    s["ids"] = torch.zeros(3, dtype=torch.int64, device="cuda")
    got = ops.low_rank_add(s["base"], s["x"], a, b, s["scales"].expand(bank, 1).contiguous(), s["ids"] + bank - 1, [n])
    check(got, s)


@pytest.mark.parametrize("m", [4, 90])
def test_captured_replayed_and_on_two_streams(m):
    s = make(m, 1024, (256, 128), 16, 4, seed=1)
    t = make(m, 1024, (256, 128), 16, 4, seed=2)
    want = [call(s), call(t)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for st, q in zip(streams, (s, t)):
        st.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(call(q))
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
    new = make(m, 1024, (256, 128), 16, 4, seed=5)          # new values in the captured inputs
    for name in ("x", "base", "a", "b", "scales", "ids"):
        s[name].copy_(new[name])
    graphs[0].replay()
    torch.cuda.synchronize()
    check(outs[0], s)
