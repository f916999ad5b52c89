"""The paged cache on the GPU against its plain form (whole numbers exactly, the others in 64 bits), each operator alone and the
three together as a serving step uses them.

Tolerances.  bf16 rounds by at most half a step, 2^-8 of the value; fp32 by 2^-24.
* Head norms and rotation: one bf16 rounding of a c - b s; the terms come from a dozen fp32 operations, so 2^-18 of the terms'
  magnitudes covers them: |y - y64| <= 2^-8 |y64| + 2^-18 (|a c| + |b s|).
* Attention: with w_j the weights of a query, A = sum w_j |v_j|.  The unnormalised weights are rounded to bf16 before their
  product with the values (2^-8 A), scores are fp32 sums of D <= 256 exact products of N(0, 1) values: their error is at
  most D 2^-23 sum |q k| / sqrt(D), about 256 * 1.2e-7 * 163 / 16 = 3.1e-4 in the exponent, on both sides of the division
  6.2e-4 A <= 2^-10 A; the result is rounded to bf16: |y - y64| <= (2^-8 + 2^-10) A + 2^-8 |y64|."""

import pytest
import torch

from oracle import paged_ref as ref

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------------------------------------------------ page plan
def _state(lens, page, width, spare, seed):
    """Tables that hold the given lengths in pages of any order, the others free."""
    held = [ref.pages(n, page) for n in lens]
    pages = torch.randperm(sum(held) + spare, generator=_gen(seed), device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -7, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = pages[at : at + n]
        at += n
    free = torch.full_like(pages, -9)
    free[:spare] = pages[at:]
    return _i32(lens), table, free, _i32([spare])


PLANS = {
    "one": dict(lens=[0], new=[1], gone=None, page=16, width=1, spare=1, rows=1),
    "nothing new": dict(lens=[5, 0, 33], new=[0, 0, 0], gone=None, page=16, width=3, spare=0, rows=0),
    "page borders": dict(lens=[15, 16, 17, 31, 32], new=[1, 1, 1, 2, 0], gone=None, page=16, width=3, spare=4, rows=9),
    "rows change hands": dict(lens=[40, 7, 64, 0], new=[3, 50, 1, 20], gone=[True, False, True, True], page=16, width=5, spare=2, rows=80),
    "all leave": dict(lens=[40, 7, 64], new=[0, 0, 0], gone=[True] * 3, page=32, width=2, spare=0, rows=5),
    "to the last page": dict(lens=[16, 16], new=[16, 32], gone=[False, True], page=16, width=2, spare=2, rows=48),
    "long": dict(lens=[0, 100001, 3], new=[70000, 1, 5000], gone=[False, False, True], page=64, width=1600, spare=1400, rows=75010),
    "one page short": dict(lens=[16, 16], new=[16, 32], gone=[False, True], page=16, width=2, spare=1, rows=48),
    "far too short": dict(lens=[0, 0], new=[1000, 1], gone=None, page=16, width=70, spare=3, rows=1001),
    "row too narrow": dict(lens=[31], new=[2], gone=None, page=16, width=2, spare=9, rows=2),
    "too many tokens": dict(lens=[0, 0], new=[3, 3], gone=None, page=16, width=2, spare=9, rows=5),
    "negative length": dict(lens=[0, 3], new=[3, -1], gone=None, page=16, width=2, spare=9, rows=5),
}


def _plan_case(name):
    if name in PLANS:
        return PLANS[name]
    b = int(name.split()[1])
    g = torch.Generator().manual_seed(b)
    pick = lambda hi: torch.randint(0, hi, (b,), generator=g).tolist()  # noqa: E731
    lens, new, gone = pick(70), pick(40), [x == 0 for x in pick(4)]
    return dict(lens=lens, new=new, gone=gone, page=16, width=9, spare=4 * b, rows=sum(new) + 3)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", [*PLANS, "random 31", "random 257", "random 1025", "random 8192"])
def test_page_plan(name, in_place):
    from tybok_b200 import ops

    c = _plan_case(name)
    lens, table, free, count = _state(c["lens"], c["page"], c["width"], c["spare"], 1)
    new, gone = _i32(c["new"]), None if c["gone"] is None else torch.tensor(c["gone"], device="cuda")
    want = ref.page_plan(lens, new, table, free, count, tokens=c["rows"], page_size=c["page"], finished=gone)
    before = [t.clone() for t in (lens, table, free, count)]
    plan = (ops.page_plan_ if in_place else ops.page_plan)(lens, new, table, free, count, tokens=c["rows"], page_size=c["page"], finished=gone)
    for field, got, w in zip(plan._fields, plan, want):
        assert got.tolist() == w, field
    if in_place:
        assert plan.block_table is table and plan.free_pages is free
    else:
        assert all(torch.equal(a, b) for a, b in zip(before, (lens, table, free, count)))


def test_page_plan_overflowing_sums_are_refused():
    from tybok_b200 import ops

    b = 64  # 64 * (2^31 - 1) tokens: their 32-bit sum would be small
    plan = ops.page_plan(_i32([0] * b), _i32([2**31 - 1] * b), torch.zeros(b, 4, dtype=torch.int32, device="cuda"), _i32([0] * 9), _i32([9]),
                         tokens=100, page_size=16)
    assert plan.missing.tolist() == [-1] and plan.free_count.tolist() == [9] and set(plan.slots.tolist()) == {-1}
    for count in (-1, 10):  # a count that no stack of nine pages has
        assert ops.page_plan(_i32([0]), _i32([1]), _i32([[0]]), _i32([0] * 9), _i32([count]), tokens=1, page_size=16).missing.tolist() == [-1]


@pytest.mark.parametrize("total", [37 * 8, 37 * 4])
def test_pages_are_neither_lost_nor_shared_over_many_steps(total):
    from tybok_b200 import ops

    b, page, width = 37, 16, 12
    g = torch.Generator().manual_seed(5)
    lens, table, free, count = _state([0] * b, page, width, total, 2)
    refused = 0
    for step in range(60):
        new = torch.randint(0, 30, (b,), generator=g) * (torch.rand(b, generator=g) < 0.5)
        gone = (torch.rand(b, generator=g) < 0.15) | (lens.cpu() + new > width * page)
        new = new.to("cuda", torch.int32)
        plan = ops.page_plan_(lens, new, table, free, count, tokens=30 * b, page_size=page, finished=gone.cuda())
        refused += plan.missing.item() != 0
        held = [t for row, n in zip(table.tolist(), lens.tolist()) for t in row[: ref.pages(n, page)]]
        assert sorted(held + free[: count.item()].tolist()) == list(range(total)), step
    assert refused < 60 and (refused > 0) == (total == 37 * 4)  # the small pool runs short at times


# ------------------------------------------------------------------------------------------------- norms, rotation, store
def _tables(n, r):
    angle = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(r // 2, device="cuda") / (r // 2))
    return angle.cos().float(), angle.sin().float()


def _pool(n, g, page, d, seed, layout="heads first"):
    x = torch.randn(n * g * page * d, generator=_gen(seed), device="cuda").to(torch.bfloat16)
    if layout == "rows first":
        return x.view(n, page, g, d).transpose(1, 2)
    if layout == "keys and values together":  # half of a wider pool
        return torch.cat([x.view(n, 1, g, page, d)] * 2, dim=1)[:, 1]
    return x.view(n, g, page, d)


@pytest.mark.parametrize("t,h,g,d,r,page,layout", [
    (1, 8, 1, 256, 256, 16, "heads first"), (33, 8, 1, 256, 256, 16, "rows first"), (5, 1, 1, 128, 128, 32, "heads first"),
    (130, 16, 16, 128, 128, 64, "heads first"), (77, 12, 4, 128, 32, 16, "keys and values together"), (64, 3, 1, 256, 144, 128, "heads first"),
    (9, 5, 5, 256, 16, 16, "rows first"), (700, 32, 8, 128, 128, 32, "keys and values together"), (4097, 2, 1, 128, 96, 16, "heads first")])
@pytest.mark.parametrize("paired", [False, True])
@pytest.mark.parametrize("normed", [True, False])
def test_head_norm_rope_store(t, h, g, d, r, page, layout, paired, normed):
    from tybok_b200 import ops

    gen = _gen(t + d)
    n_pages = ref.pages(t, page) + 3
    qkv = (torch.randn(t, (h + 2 * g) * d + 16, generator=gen, device="cuda") * 3).to(torch.bfloat16)[:, 8:-8]  # rows of a wider tensor
    qkv[t // 2] = 0  # a row whose norm divides by sqrt(eps)
    slots = torch.randperm(n_pages * page, generator=gen, device="cuda")[:t].to(torch.int32)
    slots[::7] = -1 - slots[::7]
    pos = torch.randint(0, 500, (t,), generator=gen, device="cuda").to(torch.int32)
    cos, sin = _tables(500, r)
    wq, wk = (1 + 0.3 * torch.randn(d, generator=gen, device="cuda") for _ in "qk") if normed else (None, None)
    kp, vp = _pool(n_pages, g, page, d, 1, layout), _pool(n_pages, g, page, d, 2, layout)
    k0, v0 = kp.clone(), vp.clone()
    q = ops.head_norm_rope_store(qkv, pos, slots, cos, sin, kp, vp, heads=h, norm_q=wq, norm_k=wk, eps=1e-5, paired=paired)
    ops.check_status()
    x = qkv.reshape(t, h + 2 * g, d)

    def check(got, part, weight):
        want, size = ref.head_norm_rope(part, pos, cos, sin, weight, 1e-5, paired)
        assert got.shape == want.shape and bool(((got.double() - want).abs() <= 2.0**-8 * want.abs() + 2.0**-18 * size).all())

    check(q.view(t, h, d), x[:, :h], wq)
    there = slots >= 0
    at = slots[there].long()
    got_k, got_v = kp[at // page, :, at % page], vp[at // page, :, at % page]
    full = torch.zeros(t, g, d, dtype=torch.bfloat16, device="cuda")
    full[there] = got_k
    want_k, size_k = ref.head_norm_rope(x[:, h : h + g], pos, cos, sin, wk, 1e-5, paired)
    assert bool(((full.double() - want_k).abs() <= 2.0**-8 * want_k.abs() + 2.0**-18 * size_k)[there].all())
    assert torch.equal(got_v, x[there, h + g :])
    # all other rows are as they were
    k0[at // page, :, at % page], v0[at // page, :, at % page] = got_k, got_v
    assert torch.equal(kp, k0) and torch.equal(vp, v0)


def test_store_leaves_out_what_lies_outside():
    from tybok_b200 import _lib, ops

    d, page = 128, 16
    qkv = torch.randn(6, 3 * d, generator=_gen(0), device="cuda").to(torch.bfloat16)
    cos, sin = _tables(40, d)
    for pos, slots in (([0, 1, 2, 3, 4, 40], [0, 1, 2, 3, 4, 5]), ([0, -1, 2, 3, 4, 5], [0, 1, 2, 3, 4, 5]), ([0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 4, 32])):
        kp, vp = _pool(2, 1, page, d, 3), _pool(2, 1, page, d, 4)
        k0, v0 = kp.clone(), vp.clone()
        q = ops.head_norm_rope_store(qkv, _i32(pos), _i32(slots), cos, sin, kp, vp, heads=1)
        with pytest.raises(_lib.TybokError, match="out of range"):
            ops.check_status()
        bad = [i for i in range(6) if not 0 <= pos[i] < 40 or slots[i] >= 32]
        good = [i for i in range(6) if i not in bad]
        assert torch.equal(vp[0, 0, good], qkv[good, 2 * d :])
        assert torch.equal(kp[0, 0, 6:], k0[0, 0, 6:]) and torch.equal(kp[1], k0[1]) and torch.equal(vp[1], v0[1])
        for i in bad:
            if i < 6 and slots[i] < 6:
                assert torch.equal(kp[0, 0, slots[i]], k0[0, 0, slots[i]]) and torch.equal(vp[0, 0, slots[i]], v0[0, 0, slots[i]])
            assert not bool(q[i].any()) or 0 <= pos[i] < 40
    ops.check_status()  # the word is clear again


def test_store_of_no_token_and_empty_calls():
    from tybok_b200 import ops

    kp, vp = _pool(2, 1, 16, 128, 3), _pool(2, 1, 16, 128, 4)
    cos, sin = _tables(4, 128)
    e = torch.zeros(0, 3 * 128, dtype=torch.bfloat16, device="cuda")
    assert ops.head_norm_rope_store(e, _i32([]), _i32([]), cos, sin, kp, vp, heads=1).shape == (0, 128)
    y, _ = ops.paged_attention(e[:, :128], kp, vp, _i32([[0]]), _i32([0, 0]), _i32([3]), scale=0.1, causal=True)
    assert y.shape == (0, 128)


# ------------------------------------------------------------------------------------------------------------- attention
def _attention_inputs(lens, new, h, g, d, page, seed, layout="heads first", garbage=True, tail=0, ld_q=0):
    gen = _gen(seed)
    held = [ref.pages(n, page) for n in lens]
    n_pages, width = sum(held) + 2, max(1, max(held)) + 1
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), n_pages - 1, dtype=torch.int32, device="cuda")
    kp, vp = _pool(n_pages, g, page, d, seed + 1, layout), _pool(n_pages, g, page, d, seed + 2, layout)
    used = torch.zeros(n_pages, page, dtype=torch.bool, device="cuda")
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at : at + n]
        at += n
        for j in range(n):
            used[table[b, j].item(), : max(0, min(page, lens[b] - j * page))] = True
    if garbage:  # whatever lies behind a request's last key must not get into a result
        kp.masked_fill_(~used[:, None, :, None], float("nan"))
        vp.masked_fill_(~used[:, None, :, None], float("inf"))
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + tail, h * d + ld_q, generator=gen, device="cuda").to(torch.bfloat16)[:, : h * d]
    return q, kp, vp, table, _i32(cu), _i32(lens)


def _check_attention(args, scale, causal, **kw):
    from tybok_b200 import ops

    y, planes = ops.paged_attention(*args, scale=scale, causal=causal, **kw)
    ops.check_status()
    want, size = ref.paged_attention(*args, scale=scale, causal=causal)
    err, bound = (y.double() - want).abs(), (2.0**-8 + 2.0**-10) * size + 2.0**-8 * want.abs()
    assert bool((err <= bound).all()), f"{float((err - bound).max()):.2e} over, at {torch.nonzero(err > bound)[:4].tolist()}"
    return y, planes


ATTENTION = [
    # lens, new tokens, heads, key heads, head dim, page
    ([1], [1], 1, 1, 128, 16), ([1], [1], 8, 1, 256, 16), ([17, 1, 300], [1, 1, 1], 8, 1, 256, 16),
    ([64, 65, 63, 128, 129], [1, 1, 1, 1, 1], 32, 8, 128, 32), ([700, 15], [1, 1], 16, 16, 128, 64), ([5000], [1], 8, 1, 256, 128),
    ([9000, 3, 260], [1, 1, 1], 6, 2, 256, 16), ([500] * 40, [1] * 40, 4, 1, 128, 16), ([333, 90], [2, 3], 10, 2, 128, 16),
    ([50, 300, 594], [50, 50, 50], 8, 1, 256, 64), ([130], [130], 4, 2, 256, 16), ([401, 968, 77], [401, 968, 77], 8, 1, 256, 32),
    ([1200, 64, 1, 700], [300, 64, 1, 1], 16, 16, 128, 16), ([2100], [2100], 2, 1, 128, 64), ([257, 513], [129, 255], 12, 4, 128, 32),
    ([1000, 40, 0], [128, 40, 0], 32, 8, 128, 128), ([300, 5], [17, 5], 40, 1, 128, 16), ([77, 600], [31, 200], 3, 1, 256, 512),
    ([64, 64], [0, 64], 1, 1, 128, 16), ([90], [60], 64, 1, 128, 32), ([400, 200], [4, 30], 128, 1, 128, 16), ([200], [9], 130, 1, 128, 16),
]


@pytest.mark.parametrize("lens,new,h,g,d,page", ATTENTION)
@pytest.mark.parametrize("causal", [True, False])
def test_paged_attention(lens, new, h, g, d, page, causal):
    args = _attention_inputs(lens, new, h, g, d, page, seed=sum(lens) + d)
    _check_attention(args, d**-0.5, causal)


@pytest.mark.parametrize("lens,new,h,g,d,page", [ATTENTION[2], ATTENTION[3], ATTENTION[9], ATTENTION[12], ATTENTION[14]])
@pytest.mark.parametrize("layout", ["rows first", "keys and values together"])
def test_paged_attention_layouts_planes_and_padding_rows(lens, new, h, g, d, page, layout):
    args = _attention_inputs(lens, new, h, g, d, page, seed=7, layout=layout, tail=37, ld_q=24)
    y, planes = _check_attention(args, d**-0.5, True, out_planes=True, out_shift=6, max_tokens=max(new))
    assert not bool(y[sum(new) :].any()) and not bool(planes[:, sum(new) :].any())
    got, want = planes.view(torch.float8_e5m2).float().sum(0), y.float() * 64.0
    inside = (want.abs() >= 2.0**-7) | (want == 0)
    assert torch.equal(got[inside], want[inside]) and float((got - want).abs().max()) <= 2.0**-16
    from tybok_b200 import ops

    again, only = ops.paged_attention(*args, scale=d**-0.5, causal=True, out_bf16=False, out_planes=True, out_shift=6, max_tokens=max(new))
    assert again.numel() == 0 and torch.equal(only, planes)  # same bits every time


@pytest.mark.parametrize("d,h,g", [(128, 4, 2), (256, 8, 1)])
@pytest.mark.parametrize("new", [[5, 40, 3], [200, 300, 7]])
def test_queries_that_see_no_key_give_zero(d, h, g, new):
    """More queries than keys: the first ones lie before the first key.  And requests whose cache is empty."""
    args = _attention_inputs([2, 33, 0], new, h, g, d, 16, seed=3)
    y, _ = _check_attention(args, d**-0.5, True)
    assert not bool(y[: new[0] - 2].any()) and not bool(y[new[0] + new[1] :].any())
    _check_attention(args, d**-0.5, False)


@pytest.mark.parametrize("scale", [0.0, -0.11, 3.0])
@pytest.mark.parametrize("new", [[1, 1], [70, 140]])
def test_scales_of_every_sign(scale, new):
    args = _attention_inputs([200, 333], new, 4, 2, 128, 16, seed=5)
    if scale == 3.0:  # scores of a few units all the same
        args[0].mul_(0.03)
    _check_attention(args, scale, True)


@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("d", [128, 256])
def test_scores_far_apart_and_large(new, d):
    """Rows whose scores rise by hundreds from key to key: the running maximum moves in every block."""
    q, kp, vp, table, cu, lens = _attention_inputs([900], [new], 2, 1, d, 16, seed=9)
    q.zero_()
    q.view(new, 2, d)[:, :, 0] = 8.0
    at = torch.arange(900, device="cuda")
    kp[table[0, at // 16].long(), 0, at % 16, 0] = (at.float() * 8).to(torch.bfloat16)  # scores grow by 64 a key
    from tybok_b200 import ops

    y, _ = ops.paged_attention(q, kp, vp, table, cu, lens, scale=1.0, causal=True)
    ops.check_status()
    want, size = ref.paged_attention(q, kp, vp, table, cu, lens, scale=1.0, causal=True)
    # scores are exact (one product of bf16 numbers): only the weights' and the result's rounding are left
    assert bool(((y.double() - want).abs() <= (2.0**-8 + 2.0**-16) * size + 2.0**-8 * want.abs()).all())


def test_attention_reports_indexes_out_of_range():
    from tybok_b200 import _lib, ops

    for new in ([1, 1], [40, 150]):
        q, kp, vp, table, cu, lens = _attention_inputs([100, 200], new, 4, 2, 128, 16, seed=11, garbage=False)
        good, _ = ops.paged_attention(q, kp, vp, table, cu, lens, scale=0.1, causal=True)
        ops.check_status()
        for what in ("page behind the pool", "negative page", "length", "tokens"):
            t2, l2, c2 = table.clone(), lens.clone(), cu.clone()
            if what == "page behind the pool":
                t2[1, 3] = kp.shape[0]
            elif what == "negative page":
                t2[1, 0] = -1
            elif what == "length":
                l2[1] = table.shape[1] * 16 + 1
            else:
                c2[2] = q.shape[0] + 5
            y, _ = ops.paged_attention(q, kp, vp, t2, c2, l2, scale=0.1, causal=True)
            with pytest.raises(_lib.TybokError, match="out of range"):
                ops.check_status()
            assert torch.equal(y[: new[0]], good[: new[0]])  # the other request is untouched
    ops.check_status()


def test_a_hint_that_is_too_small_changes_no_more_than_rounding():
    args = _attention_inputs([1000, 90], [130, 70], 8, 2, 128, 16, seed=13)
    for most in (1, 16, 200):
        _check_attention(args, 128**-0.5, True, max_tokens=most)


# ---------------------------------------------------------------------------------------------------- together, and graphs
@pytest.mark.parametrize("h,g,d,page,causal", [(8, 1, 256, 16, False), (12, 4, 128, 32, True)])
def test_a_serving_loop_equals_whole_sequences(h, g, d, page, causal):
    """Requests come, bring prompts and single tokens, and leave; their rows and pages go to others.  Every step's output is
    that of attention over the request's whole sequence so far, from keys and values that were never in a cache."""
    from tybok_b200 import ops

    b, width, total, rows = 6, 40, 6 * 20, 700
    gen, rng = _gen(1), torch.Generator().manual_seed(1)
    lens, table, free, count = _state([0] * b, page, width, total, 3)
    kp = torch.full((total, g, page, d), float("nan"), dtype=torch.bfloat16, device="cuda")
    vp = kp.clone()
    cos, sin = _tables(1024, d)
    wq, wk = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda") for _ in "qk")
    history = [[] for _ in range(b)]
    for step in range(12):
        new = [int(torch.randint(1, 150, (1,), generator=rng)) if step % 4 == 0 else int(torch.randint(0, 3, (1,), generator=rng)) for _ in range(b)]
        gone = [step > 0 and (float(torch.rand(1, generator=rng)) < 0.2 or step % 4 == 0 and len(history[i]) > 200) for i in range(b)]
        qkv = torch.randn(rows, (h + 2 * g) * d, generator=gen, device="cuda").to(torch.bfloat16)
        plan = ops.page_plan_(lens, _i32(new), table, free, count, tokens=rows, page_size=page, finished=torch.tensor(gone, device="cuda"))
        q = ops.head_norm_rope_store(qkv, plan.pos, plan.slots, cos, sin, kp, vp, heads=h, norm_q=wq, norm_k=wk)
        y, _ = ops.paged_attention(q, kp, vp, plan.block_table, plan.cu_tokens, plan.key_lens, scale=d**-0.5, causal=causal)
        ops.check_status()
        assert plan.missing.item() == 0 and not bool(y[sum(new) :].any())
        at = 0
        for i in range(b):
            if gone[i]:
                history[i] = []
            history[i] += list(qkv[at : at + new[i]].unbind(0))
            if new[i]:
                x = torch.stack(history[i]).view(-1, h + 2 * g, d)
                n = x.shape[0]
                pos = torch.arange(n, device="cuda")
                turn = lambda part, w: ref.head_norm_rope(part, pos, cos, sin, w, 1e-6, False)[0].to(torch.bfloat16)  # noqa: E731
                # one page that holds the whole sequence
                k, v = turn(x[:, h : h + g], wk).transpose(0, 1)[None], x[:, h + g :].transpose(0, 1)[None]
                want, size = ref.paged_attention(turn(x[:, :h], wq)[n - new[i] :].reshape(new[i], h * d), k, v,
                                                 torch.zeros(1, 1, dtype=torch.int32, device="cuda"), _i32([0, new[i]]), _i32([n]),
                                                 scale=d**-0.5, causal=causal)
                # beside the bound of the attention: a query or key that lies next to a rounding border may have been rounded to
                # the other side, a step of 2^-7 in single factors of the scores
                err = (y[at : at + new[i]].double() - want).abs()
                assert bool((err <= (2.0**-8 + 2.0**-10 + 2.0**-7) * size + 2.0**-8 * want.abs()).all()), (step, i)
            at += new[i]


def test_two_captured_steps_replay_in_turn():
    """The three calls as a graph in place, captured twice on the same state and replayed in turn, against the same steps run eagerly."""
    from tybok_b200 import ops

    h, g, d, page, b, rows = 8, 2, 128, 16, 5, 24
    gen = _gen(4)
    cos, sin = _tables(256, d)
    steps = [(torch.randint(0, 4, (b,), generator=gen, device="cuda").to(torch.int32),
              torch.rand(b, generator=gen, device="cuda") < 0.2,
              torch.randn(rows, (h + 2 * g) * d, generator=gen, device="cuda").to(torch.bfloat16)) for _ in range(6)]

    def fresh():
        kp, vp = _pool(30, g, page, d, 5), _pool(30, g, page, d, 6)
        return _state([20, 3, 31, 0, 16], page, 6, 18, 7) + (kp, vp)

    def step(state, new, gone, qkv):
        lens, table, free, count, kp, vp = state
        plan = ops.page_plan_(lens, new, table, free, count, tokens=rows, page_size=page, finished=gone)
        q = ops.head_norm_rope_store(qkv, plan.pos, plan.slots, cos, sin, kp, vp, heads=h)
        return ops.paged_attention(q, kp, vp, table, plan.cu_tokens, lens, scale=d**-0.5, causal=True, max_tokens=4)[0]

    eager = fresh()
    want = [step(eager, *s).clone() for s in steps]
    state = fresh()
    keep = [t.clone() for t in state]
    new, gone, qkv = (t.clone() for t in steps[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state, new, gone, qkv)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(state, new, gone, qkv))
        graphs.append(graph)
    for t, k in zip(state, keep):
        t.copy_(k)
    for i, s in enumerate(steps):
        for dst, src in zip((new, gone, qkv), s):
            dst.copy_(src)
        graphs[i & 1].replay()
        assert torch.equal(outs[i & 1], want[i]), i
    assert all(torch.equal(a, b) for a, b in zip(state, eager))
    ops.check_status()


def test_on_another_stream_than_the_default():
    from tybok_b200 import ops

    args = _attention_inputs([900, 40], [1, 1], 8, 1, 256, 16, seed=21)
    want = ops.paged_attention(*args, scale=0.06, causal=True)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.paged_attention(*args, scale=0.06, causal=True)[0] for _ in range(20)]
    other = [ops.paged_attention(*args, scale=0.06, causal=True)[0] for _ in range(20)]  # at the same time
    torch.cuda.synchronize()
    assert all(torch.equal(want, y) for y in got + other)
