"""Norms and rotation of query and key heads, and their store into pages, against the definition in 64 bits.

Bound of an output value: half a step of bf16 (2^-8 of it), and for the arithmetic in 32 bits a few steps of 2^-24 of the absolute terms u_i |cos| + u_j |sin|: the mean square (up to 512
additions, but their errors are relative to a sum of squares: 2^-15 at most, half of that after the root), the products, and sine and cosine of a fraction of a turn
held in 24 bits, off by 2^-22 of a radian's multiple at most.  2^-13 covers them."""
import math

import pytest
import torch

from hyperqwen_rtx4080s32_b200 import ops

pytestmark = pytest.mark.gpu


def bf16(*shape, seed, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(torch.bfloat16)


def make(t, hq, hk, d, rot, gated=False, far=1 << 20, norm=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    inv, amp = ops.rotary_frequencies(rot, 1e6, scaling="yarn" if rot >= 32 else None, factor=8, original_context=32768)
    return dict(qkv=bf16(t, (2 if gated else 1) * hq * d + 2 * hk * d, seed=seed + 1, std=2.0), positions=torch.randint(0, far, (t,), device="cuda", generator=g), inv_freq=inv,
                n_heads=hq, n_kv_heads=hk, head_dim=d), dict(q_norm=1 + bf16(d, seed=seed + 2, std=0.2) if norm else None,
                                                             k_norm=1 + bf16(d, seed=seed + 3, std=0.2) if norm else None, amplitude=amp, gated=gated)


def want_of(s, how, interleaved=False, eps=1e-6):
    """[(values, absolute terms)] of q and k, and v."""
    hq, hk, d = s["n_heads"], s["n_kv_heads"], s["head_dim"]
    w = (2 if how["gated"] else 1) * d
    q, k, v = s["qkv"].double().split((hq * w, hk * d, hk * d), dim=1)
    angle = (s["positions"].double()[:, None] * s["inv_freq"])[:, None, :]
    cos, sin = angle.cos() * how["amplitude"], angle.sin() * how["amplitude"]
    out, half = [], s["inv_freq"].numel()
    for x, weight in ((q.unflatten(1, (hq, w))[..., :d], how["q_norm"]), (k.unflatten(1, (hk, d)), how["k_norm"])):
        u = x.clone() if weight is None else x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
        size = u.abs()
        i = torch.arange(half, device="cuda")
        i, j = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        one, two, a, b = u[..., i], u[..., j], size[..., i], size[..., j]
        u[..., i], u[..., j] = one * cos - two * sin, two * cos + one * sin
        size[..., i], size[..., j] = a * cos.abs() + b * sin.abs(), b * cos.abs() + a * sin.abs()
        out.append((u, size))
    return out, v.unflatten(1, (hk, d))


def near(got, want):
    err = (got.double() - want[0]).abs()
    bound = 2.0 ** -8 * want[0].abs() + 2.0 ** -13 * want[1]
    assert bool((err <= bound).all()), f"worst {float((err / bound.clamp_min(1e-30)).max()):.3g} of the bound"


CASES = [(1, 1, 1, 8, 0, False), (1, 40, 8, 128, 128, False), (3, 2, 1, 8, 8, True), (5, 3, 3, 16, 6, False), (17, 5, 1, 64, 64, True), (9, 4, 2, 72, 24, False), (4, 7, 2, 80, 32, True),
         (33, 24, 4, 256, 64, True), (2, 3, 1, 512, 512, False), (130, 6, 2, 96, 96, True), (700, 40, 8, 128, 64, False), (5, 2, 2, 256, 250, False), (3, 1, 1, 128, 2, True), (6, 70, 3, 64, 16, False)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_the_definition(case, interleaved):
    t, hq, hk, d, rot, gated = case
    for norm in (True, False):
        s, how = make(t, hq, hk, d, rot, gated, norm=norm, seed=d + rot)
        (q, k), _ = want_of(s, how, interleaved)
        got = ops.qk_norm_rope(**s, **how, interleaved=interleaved)
        assert got[0].shape == (t, hq, d) and got[1].shape == (t, hk, d)
        near(got[0], q)
        near(got[1], k)
        again = ops.qk_norm_rope(**dict(s, positions=s["positions"].int()), **how, interleaved=interleaved)
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


def test_positions_that_are_far_and_negative():
    s, how = make(4, 2, 1, 128, 128, seed=3)
    s["positions"] = torch.tensor([0, 10_000_000, (1 << 31) + 5, -77], device="cuda")
    (q, k), _ = want_of(s, how)
    # 64 bits of angle: 2^31 radians leave 2^-22 of one in the definition itself
    got = ops.qk_norm_rope(**s, **how)
    near(got[0], q)
    near(got[1], k)


def test_one_norm_only_small_heads_and_another_eps():
    s, how = make(3, 4, 2, 64, 32, seed=9)
    s["qkv"] *= 2.0 ** -12                   # the mean square is as small as eps
    for q_norm, k_norm in ((how["q_norm"], None), (None, how["k_norm"])):
        h = dict(how, q_norm=q_norm, k_norm=k_norm)
        (q, k), _ = want_of(s, h, eps=1e-5)
        got = ops.qk_norm_rope(**s, **h, eps=1e-5)
        near(got[0], q)
        near(got[1], k)
    s["qkv"].zero_()
    assert all(bool((x == 0).all()) for x in ops.qk_norm_rope(**s, **how))


def pages_of(n, rows, heads, d, head_major, seed):
    return bf16(n, heads, rows, d, seed=seed).transpose(1, 2) if head_major else bf16(n, rows, heads, d, seed=seed)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("case,rows,head_major", [((1, 40, 8, 128, 128, False), 16, True), ((19, 24, 4, 256, 64, True), 16, False), ((50, 3, 2, 72, 16, False), 5, True), ((300, 5, 1, 64, 64, True), 64, False),
                                                  ((7, 2, 2, 8, 8, False), 1, True)], ids=str)
def test_store(case, rows, head_major, wide):
    t, hq, hk, d, rot, gated = case
    s, how = make(t, hq, hk, d, rot, gated, seed=4)
    n = -(-t // rows) + 3
    k_pages, v_pages = pages_of(n, rows, hk, d, head_major, 31), pages_of(n, rows, hk, d, not head_major, 32)
    before = [k_pages.clone(), v_pages.clone()]
    slots = torch.randperm(n * rows, generator=torch.Generator().manual_seed(t))[:t].cuda()
    if t > 2:
        slots[1], slots[2] = -1, -7
    if not wide:
        slots = slots.int()
    q = ops.qk_norm_rope_store(**s, k_pages=k_pages, v_pages=v_pages, slots=slots, **how)
    plain_q, plain_k = ops.qk_norm_rope(**s, **how)
    _, v = want_of(s, how)
    assert torch.equal(q, plain_q)
    for tok, slot in enumerate(slots.tolist()):
        if slot >= 0:
            before[0][slot // rows, slot % rows], before[1][slot // rows, slot % rows] = plain_k[tok], v[tok].to(torch.bfloat16)
    assert torch.equal(k_pages, before[0]) and torch.equal(v_pages, before[1])
    assert ops.device_status() == 0


def test_a_slot_beyond_the_cache_stores_nothing_and_is_reported():
    s, how = make(5, 2, 1, 64, 64)
    k_pages, v_pages = pages_of(3, 4, 1, 64, True, 1), pages_of(3, 4, 1, 64, True, 2)
    before = [k_pages.clone(), v_pages.clone()]
    q = ops.qk_norm_rope_store(**s, k_pages=k_pages, v_pages=v_pages, slots=torch.tensor([12, 13, 1 << 40, -1, -(1 << 40)], device="cuda"), **how)
    assert torch.equal(q, ops.qk_norm_rope(**s, **how)[0])
    assert torch.equal(k_pages, before[0]) and torch.equal(v_pages, before[1])
    assert ops.device_status() == 2 and ops.device_status() == 0


def test_rows_that_start_anywhere_and_values_that_are_not_finite():
    s, how = make(6, 3, 1, 128, 64, seed=8)
    want = ops.qk_norm_rope(**s, **how)
    buf = torch.zeros(6, s["qkv"].shape[1] + 9, dtype=torch.bfloat16, device="cuda")
    view = buf[:, 3:3 + s["qkv"].shape[1]]
    view.copy_(s["qkv"])
    for got, w in zip(ops.qk_norm_rope(**dict(s, qkv=view), **how), want):
        assert torch.equal(got, w)
    s["qkv"][2, 130] = float("inf")           # second head of the third token
    got = ops.qk_norm_rope(**s, **how)
    assert torch.equal(got[1], want[1])
    ok = torch.ones(6, 3, dtype=torch.bool, device="cuda")
    ok[2, 1] = False
    assert torch.equal(got[0][ok], want[0][ok]) and bool(got[0][2, 1].isnan().any())


def test_captured_replayed_and_on_another_stream():
    s, how = make(9, 6, 2, 128, 128, seed=6)
    k_pages, v_pages = pages_of(4, 16, 2, 128, True, 1), pages_of(4, 16, 2, 128, True, 2)
    slots = torch.arange(9, device="cuda") + 20
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=st):
        q = ops.qk_norm_rope_store(**s, k_pages=k_pages, v_pages=v_pages, slots=slots, **how)
    new, _ = make(9, 6, 2, 128, 128, seed=60)
    s["qkv"].copy_(new["qkv"])
    s["positions"].copy_(new["positions"])
    slots += 3
    g.replay()
    torch.cuda.synchronize()
    want_q, want_k = ops.qk_norm_rope(**s, **how)
    assert torch.equal(q, want_q) and torch.equal(k_pages.transpose(1, 2).transpose(1, 2).reshape(64, 2, 128)[23:32], want_k)


def test_frequencies():
    inv, amp = ops.rotary_frequencies(64, 1e4, device="cpu")
    assert inv.dtype == torch.float64 and amp == 1.0 and math.isclose(float(inv[3]), 1e4 ** (-6 / 64), rel_tol=1e-15)
