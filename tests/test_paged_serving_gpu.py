"""The paged cache as a server uses it: several layers and steps through ``PagedCache``, its graph, streams at once, dispatch that others
intercept, waits that run out, and pools beyond 2^31 elements.

Tolerances are those of ``test_paged_gpu``: |y - y64| <= (2^-8 + 2^-10) sum w |v| + 2^-8 |y64| for an attention, whose keys
and values are read back from the cache where a run is checked (so that no second rounding enters)."""

import pytest
import torch
from test_dispatch_gpu import _Seen, _Sub
from test_paged_gpu import _attention_inputs, _check_attention, _gen, _i32, _tables
from test_time_outs_gpu import _runs_out

from oracle import paged_ref as ref

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:There is a performance drop")]
MMA, EPILOGUE = 102, 104  # TYBOK_DEV_TIMEOUT_*


def _cache(g, d, page, **over):
    from tybok_b200.paged import PagedCache

    return PagedCache(**{**dict(layers=2, requests=4, pages=60, page_size=page, kv_heads=g, head_dim=d, width=30), **over})


@pytest.mark.parametrize("h,g,d,page", [(8, 1, 256, 16), (12, 4, 128, 32)])
def test_layers_and_steps(h, g, d, page):
    """Prompts of different lengths, then single tokens, one request replaced by another; every layer has its own keys."""
    from tybok_b200 import ops

    cache, gen = _cache(g, d, page), _gen(1)
    cos, sin = _tables(512, d)
    steps = [([70, 0, 33, 150], [0] * 4), ([1, 1, 1, 1], [0] * 4), ([1, 0, 90, 1], [0, 0, 1, 0]), ([0, 1, 1, 1], [1, 0, 0, 0])]
    lens = [0] * 4
    for new, gone in steps:
        rows = sum(new) + 5
        plan = cache.step(_i32(new), tokens=rows, finished=torch.tensor(gone, dtype=torch.bool, device="cuda"))
        lens = [(0 if out else n) + k for n, k, out in zip(lens, new, gone)]
        assert plan.missing.item() == 0 and cache.key_lens.tolist() == lens
        for layer in range(2):
            qkv = torch.randn(rows, (h + 2 * g) * d, generator=gen, device="cuda").to(torch.bfloat16)
            y, none = cache.attend(layer, qkv, cos, sin, heads=h)
            ops.check_status()
            assert none.numel() == 0 and not bool(y[sum(new) :].any())
            x = qkv.view(rows, h + 2 * g, d)
            turn = lambda part: ref.head_norm_rope(part, plan.pos.long(), cos, sin, None, 1e-6, False)  # noqa: E731
            page_of, row_of = plan.slots[: sum(new)] // page, plan.slots[: sum(new)] % page
            k, size = turn(x[:, h : h + g])
            got = cache.k_pages[layer][page_of.long(), :, row_of.long()].double()
            assert bool(((got - k[: sum(new)]).abs() <= 2.0**-8 * k[: sum(new)].abs() + 2.0**-18 * size[: sum(new)]).all())
            assert torch.equal(cache.v_pages[layer][page_of.long(), :, row_of.long()], x[: sum(new), h + g :])
            q = ops.head_norm_rope_store(qkv, plan.pos, plan.slots, cos, sin, cache.k_pages[layer], cache.v_pages[layer], heads=h)  # the same again
            want, size = ref.paged_attention(q, cache.k_pages[layer], cache.v_pages[layer], plan.block_table, plan.cu_tokens, plan.key_lens,
                                             scale=d**-0.5, causal=True)
            assert bool(((y.double() - want).abs() <= (2.0**-8 + 2.0**-10) * size + 2.0**-8 * want.abs()).all())


def test_a_step_without_room_leaves_everything():
    from tybok_b200 import ops

    cache = _cache(2, 128, 16, pages=5, width=5)
    cos, sin = _tables(512, 128)
    qkv = torch.randn(100, 8 * 128, generator=_gen(2), device="cuda").to(torch.bfloat16)
    cache.step(_i32([20, 0, 20, 0]), tokens=100)
    cache.attend(0, qkv, cos, sin, heads=4)
    keep = [t.clone() for t in (cache.key_lens, cache.block_table, cache.free_pages, cache.free_count, cache.k_pages[0], cache.v_pages[0])]
    plan = cache.step(_i32([1, 40, 0, 0]), tokens=100)
    y, _ = cache.attend(0, qkv, cos, sin, heads=4)
    assert plan.missing.item() == 2 and not bool(y.any())
    bits = lambda t: t.view(torch.int16) if t.dtype == torch.bfloat16 else t  # noqa: E731  (pages that nobody wrote may hold NaN)
    for a, b in zip(keep, (cache.key_lens, cache.block_table, cache.free_pages, cache.free_count, cache.k_pages[0], cache.v_pages[0])):
        assert torch.equal(bits(a), bits(b))
    ops.check_status()


def test_a_captured_step_of_two_layers():
    cos, sin = _tables(256, 256)
    gen = _gen(3)
    qkv = torch.randn(2, 8, 10 * 256, generator=gen, device="cuda").to(torch.bfloat16)
    prompt = torch.randn(2, 60, 10 * 256, generator=gen, device="cuda").to(torch.bfloat16)
    new = _i32([1, 1, 0, 1])

    def begin():
        cache = _cache(1, 256, 16)
        cache.step(_i32([31, 0, 9, 16]), tokens=60)
        for layer in range(2):
            cache.attend(layer, prompt[layer], cos, sin, heads=8)
        return cache

    def step(cache):
        cache.step(new, tokens=8)
        return [cache.attend(layer, qkv[layer], cos, sin, heads=8, max_tokens=1)[0] for layer in range(2)]

    eager, cache = begin(), begin()
    want = [[y.clone() for y in step(eager)] for _ in range(20)]
    spare = begin()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(spare)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for i in range(20):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])), i
    assert torch.equal(cache.key_lens, eager.key_lens) and torch.equal(cache.block_table, eager.block_table)


def _lengths(seed):
    """Requests, heads and lengths of any kind: few and many, short and long, some without tokens or keys."""
    rng = torch.Generator().manual_seed(seed)
    pick = lambda hi: int(torch.randint(0, hi, (1,), generator=rng))  # noqa: E731
    d, g = (128, 256)[pick(2)], (1, 2, 3, 8)[pick(4)]
    h = g * (1, 2, 4, 5, 8, 16)[pick(6)]
    b = (1, 2, 3, 7, 20, 70)[pick(6)]
    keys, most = (40, 300, 2000, 6000)[pick(4)] // max(1, b // 8) + 1, (1, 3, 20, 130, 700)[pick(5)] // max(1, b // 8) + 1
    new = [pick(most + 1) for _ in range(b)]
    lens = [n + pick(keys) if pick(9) else n for n in new]
    return lens, new, h, g, d, (16, 32, 64, 128)[pick(4)], pick(2) == 0


@pytest.mark.parametrize("seed", range(40))
def test_lengths_of_any_kind(seed):
    lens, new, h, g, d, page, causal = _lengths(seed)
    args = _attention_inputs(lens, new, h, g, d, page, seed=seed, tail=seed % 3)
    y, _ = _check_attention(args, d**-0.5, causal)
    assert not bool(y[sum(new) :].any())


@pytest.mark.parametrize("lens,new,h,g,d", [([2000, 300], [128, 64], 8, 2, 128), ([900, 800], [50, 50], 8, 1, 256), ([6000], [20], 8, 1, 256),
                                            ([500] * 30, [60] * 30, 8, 1, 128), ([3000], [1], 8, 1, 256)])
def test_streams_at_once_and_the_same_bits(lens, new, h, g, d):
    """Launches with workspaces of their own run side by side; every one gives the bits of the first."""
    from tybok_b200 import ops

    args = _attention_inputs(lens, new, h, g, d, 32, seed=5)
    call = lambda: ops.paged_attention(*args, scale=d**-0.5, causal=True)[0]  # noqa: E731
    want = call()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(want, y) for y in got)
    ops.check_status()


@pytest.mark.parametrize("lens,new,h,g,d", [([2000, 300], [300, 64], 8, 2, 128), ([900, 800], [50, 50], 8, 1, 256), ([2000], [400], 8, 1, 256),
                                            ([700], [30], 16, 1, 128)])
def test_waits_that_run_out(lens, new, h, g, d):
    """Both tile forms, with parts joined in a cluster and by the second kernel."""
    from tybok_b200 import ops

    args = _attention_inputs(lens, new, h, g, d, 32, seed=6)
    _runs_out(lambda: ops.paged_attention(*args, scale=d**-0.5, causal=True)[0], (MMA, EPILOGUE))


def test_interception():
    from tybok_b200 import ops

    q, *rest = _attention_inputs([40, 9], [3, 2], 8, 1, 256, 16, seed=7)
    attend = lambda x: ops.paged_attention(x, *rest, scale=0.06, causal=True)[0]  # noqa: E731
    want = attend(q)
    with _Seen() as seen:
        y = attend(q.clone())
    assert "tybok_b200.paged_attention.default" in seen.names and torch.equal(y, want)
    z = attend(q.as_subclass(_Sub))
    assert type(z) is _Sub and torch.equal(z.as_subclass(torch.Tensor), want)
    xs = torch.stack([q, q * 2])
    assert torch.equal(torch.vmap(attend)(xs), torch.stack([attend(x) for x in xs]))

    cos, sin = _tables(64, 256)
    pool = torch.zeros(2, 4, 1, 16, 256, dtype=torch.bfloat16, device="cuda")
    qkv = torch.randn(5, 10 * 256, generator=_gen(8), device="cuda").to(torch.bfloat16)
    store = lambda x: ops.head_norm_rope_store(x, _i32([0, 1, 2, 3, 4]), _i32([0, 1, 2, 3, 40]), cos, sin, pool[0], pool[1], heads=8)  # noqa: E731
    want = store(qkv)
    kept = pool.clone()
    with _Seen() as seen:
        y = store(qkv.clone())
    assert "tybok_b200.head_norm_rope_store.default" in seen.names and torch.equal(y, want) and torch.equal(pool, kept)
    assert type(store(qkv.as_subclass(_Sub))) is _Sub

    plan = lambda x, f: f(x, _i32([1, 2]), _i32([[0, 0], [1, 0]]), _i32([2, 3, 0]), _i32([2]), tokens=3, page_size=16)  # noqa: E731
    for f, name in ((ops.page_plan, "page_plan"), (ops.page_plan_, "page_plan_")):
        want = plan(_i32([16, 4]), f)
        with _Seen() as seen:
            got = plan(_i32([16, 4]), f)
        assert f"tybok_b200.{name}.default" in seen.names and all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("d,new", [(128, [1, 200]), (256, [1, 100]), (128, [1, 2])])
def test_pools_beyond_31_bits(d, new):
    """Keys and values of a page side by side in one tensor of more than 2^31 elements; the pages in use lie at its end and its start."""
    from tybok_b200 import ops

    page, g, h = 128, 2, 8
    n_pages = (1 << 31) // (2 * g * page * d) + 7
    pool = torch.empty(n_pages, 2, g, page, d, dtype=torch.bfloat16, device="cuda")
    kp, vp = pool[:, 0], pool[:, 1]
    used = torch.tensor([n_pages - 1, 0, n_pages - 2, n_pages - 3, 1], device="cuda")
    pool[used] = torch.randn(5, 2, g, page, d, generator=_gen(9), device="cuda").to(torch.bfloat16)
    lens, table = [130, 300], torch.stack([used[:3], used[2:]]).to(torch.int32)
    cu = [0, new[0], sum(new)]
    cos, sin = _tables(512, d)
    qkv = torch.randn(cu[-1], (h + 2 * g) * d, generator=_gen(10), device="cuda").to(torch.bfloat16)
    pos = _i32([lens[b] - new[b] + i for b in range(2) for i in range(new[b])])
    owner = [b for b in range(2) for _ in range(new[b])]
    slots = _i32([int(table[b, p // page]) * page + p % page for b, p in zip(owner, pos.tolist())])
    q = ops.head_norm_rope_store(qkv, pos, slots, cos, sin, kp, vp, heads=h)
    assert torch.equal(vp[(slots // page).long(), :, (slots % page).long()], qkv.view(-1, h + 2 * g, d)[:, h + g :])
    # the pages in use alone, for the oracle
    small = pool[used].contiguous()
    where = {int(p): i for i, p in enumerate(used.tolist())}
    near = _i32([[where[int(p)] for p in row] for row in table.tolist()])
    want, size = ref.paged_attention(q, small[:, 0], small[:, 1], near, _i32(cu), _i32(lens), scale=d**-0.5, causal=True)
    y, _ = ops.paged_attention(q, kp, vp, table, _i32(cu), _i32(lens), scale=d**-0.5, causal=True)
    ops.check_status()
    assert bool(((y.double() - want).abs() <= (2.0**-8 + 2.0**-10) * size + 2.0**-8 * want.abs()).all())


@pytest.mark.parametrize("lens,new,h,g,d", [([300, 90], [130, 40], 4, 2, 128), ([200], [50], 8, 1, 256), ([90], [1], 8, 1, 256)])
def test_outputs_that_are_only_16_byte_aligned(lens, new, h, g, d):
    """The C entry point takes any output on a 16-byte boundary, and leaves the bytes around it."""
    import ctypes

    from tybok_b200 import _lib, ops

    q, kp, vp, table, cu, klen = _attention_inputs(lens, new, h, g, d, 16, seed=11)
    want, planes = ops.paged_attention(q, kp, vp, table, cu, klen, scale=0.08, causal=True, out_planes=True, out_shift=3)
    lib, n = _lib.load(), q.numel()
    out = torch.full((n + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    out_planes = torch.full((3 * n + 64,), 9, dtype=torch.uint8, device="cuda")
    need = lib.tybok_paged_attention_workspace_bytes(h, g, d, max(new))
    ws = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    strides = lambda t: (ctypes.c_int64 * 3)(*t.stride()[:3])  # noqa: E731
    rc = lib.tybok_paged_attention(q.data_ptr(), q.stride(0), kp.data_ptr(), strides(kp), vp.data_ptr(), strides(vp), table.data_ptr(), table.stride(0),
                                   cu.data_ptr(), klen.data_ptr(), out.data_ptr() + 16, out_planes.data_ptr() + 16, 3, q.shape[0], len(lens), h, g, d,
                                   kp.shape[0], 16, table.shape[1], max(new), 1, 0.08, ws.data_ptr(), need, None,
                                   torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.tybok_last_error()
    assert torch.equal(out[8 : 8 + n].view_as(want), want) and bool((out[:8] == 7).all()) and bool((out[8 + n :] == 7).all())
    assert torch.equal(out_planes[16 : 16 + 3 * n], planes.view(torch.uint8).reshape(-1))
    assert bool((out_planes[:16] == 9).all()) and bool((out_planes[16 + 3 * n :] == 9).all())


def test_plan_refuses_lengths_beyond_31_bits():
    from tybok_b200 import ops

    table, free = torch.zeros(1, 2050, dtype=torch.int32, device="cuda"), _i32([0, 1, 2, 3])
    plan = ops.page_plan(_i32([2**31 - 100]), _i32([200]), table, free, _i32([4]), tokens=200, page_size=1 << 20)
    assert plan.missing.item() == -1 and plan.key_lens.item() == 2**31 - 100 and bool((plan.slots == -1).all())


@pytest.mark.parametrize("h,g,d", [(8, 1, 256), (8, 2, 128), (1, 1, 128)])
def test_requests_that_claim_the_same_tokens_are_reported(h, g, d):
    """Bounds that go back and forth: the status word says so, rows outside the output are never touched."""
    from tybok_b200 import ops

    q, kp, vp, table, _, _ = _attention_inputs([60] * 6, [40] * 6, h, g, d, 16, seed=12)
    out = ops.paged_attention(q, kp, vp, table, _i32([0, 240, 0, 240, 0, 240, 0]), _i32([60] * 6), scale=0.1, causal=False)[0]
    torch.cuda.synchronize()
    with pytest.raises(ops._lib.TybokError, match="out of range"):
        ops.check_status()
    assert out.shape == q.shape
    y, _ = _check_attention((q, kp, vp, table, _i32([0, 40, 80, 120, 160, 200, 240]), _i32([60] * 6)), 0.1, False)  # and the next call is right
    assert y.shape == q.shape


@pytest.mark.parametrize("most_keys", [64, 200])
@pytest.mark.parametrize("tokens", [10, 3, 16])
def test_many_short_tiles_in_a_row(tokens, most_keys):
    """Hundreds of requests of one key block or a few at head_dim 256, so that a CTA's share runs through many tiles whose blocks fall to
    one group of softmax warps alone, with warps that have no query rows; the same bits from run to run."""
    from tybok_b200 import ops

    rng = torch.Generator().manual_seed(tokens + most_keys)
    lens = [int(x) for x in torch.randint(tokens, most_keys + 1, (700,), generator=rng)]
    args = _attention_inputs(lens, [tokens] * 700, 8, 1, 256, 16, seed=14)
    want, _ = _check_attention(args, 0.0625, False)
    got = [ops.paged_attention(*args, scale=0.0625, causal=False)[0] for _ in range(100)]
    ops.check_status()
    assert all(torch.equal(want, y) for y in got)


@pytest.mark.parametrize("requests", [3, 300])  # joined in clusters; a line of tiles
@pytest.mark.parametrize("blocks", [3, 4, 5, 6, 7])
def test_a_tile_ends_with_its_last_product(blocks, requests):
    """Tiles of a few key blocks at head_dim 256 with scores so alike that no output row is ever rescaled: only the end of a tile waits for
    a product.  The same bits from run to run."""
    from tybok_b200 import ops

    rng = torch.Generator().manual_seed(blocks)
    lens = [64 * blocks - int(x) for x in torch.randint(0, 30, (requests,), generator=rng)]
    args = _attention_inputs(lens, [12] * requests, 8, 1, 256, 16, seed=15)
    want, _ = _check_attention(args, 0.01, False)
    got = [ops.paged_attention(*args, scale=0.01, causal=False)[0] for _ in range(100)]
    ops.check_status()
    assert all(torch.equal(want, y) for y in got)


@pytest.mark.parametrize("in_place", [False, True])
def test_a_plan_of_the_most_token_rows(in_place):
    """2^31 - 1 token rows: the last stride of the threads over them passes 2^31."""
    from tybok_b200 import ops

    rows = 2**31 - 1
    lens, table, free, count = _i32([40]), _i32([[3, 1, 0]]), _i32([2, 5, 4]), _i32([2])
    plan = (ops.page_plan_ if in_place else ops.page_plan)(lens, _i32([7]), table, free, count, tokens=rows, page_size=16)
    assert plan.missing.tolist() == [0] and plan.cu_tokens.tolist() == [0, 7] and plan.key_lens.tolist() == [47]
    assert plan.block_table.tolist() == [[3, 1, 0]] and plan.free_pages.tolist() == [2, 5, 4] and plan.free_count.tolist() == [2]
    assert plan.pos[:8].tolist() == [*range(40, 47), 0] and plan.slots[:8].tolist() == [*range(8, 15), -1]
    for t, behind in ((plan.pos, 0), (plan.slots, -1)):
        assert t.numel() == rows and all(bool((part == behind).all()) for part in t[7:].split(1 << 28))


def test_a_request_that_grows_to_the_most_keys():
    """Lengths, positions and token numbers next to 2^31, in one request and behind others."""
    from tybok_b200 import ops

    page, top = 1 << 20, 2**31 - 1
    table = torch.arange(2 * 2048, dtype=torch.int32, device="cuda").view(2, 2048) % 2000
    plan = ops.page_plan(_i32([0, top - 3000]), _i32([5000, 3000]), table, _i32([7] * 2000), _i32([9]), tokens=8000, page_size=page)
    assert plan.missing.tolist() == [0] and plan.key_lens.tolist() == [5000, top] and plan.cu_tokens.tolist() == [0, 5000, 8000]
    assert plan.pos[5000:].tolist() == list(range(top - 3000, top))
    last = int(table[1, 2047])
    assert plan.slots[5000:].tolist() == [last * page + p % page for p in range(top - 3000, top)]


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("causal", [True, False])
def test_scores_near_the_lowest_value(d, new, causal):
    """Finite scores far below -1e30: equal ones average their values, and among unequal ones the highest alone counts.  They are single
    products of powers of two, so exact, and differ by nothing or by more than any exponential can tell: the bound of
    ``_check_attention`` holds as it is."""
    q, kp, vp, table, cu, lens = _attention_inputs([900], [new], 2, 1, d, 16, seed=16)
    q.zero_()
    q.view(new, 2, d)[:, :, 0] = 2.0**60
    at = torch.arange(900, device="cuda")
    for some in (2.0**60, 2.0**62):  # the scores of two keys of three; the others' are -2^118, -3e35
        kp[table[0, at // 16].long(), 0, at % 16] = 0
        kp[table[0, at // 16].long(), 0, at % 16, 0] = torch.where(at % 3 == 0, -(2.0**60), -some).to(torch.bfloat16)
        _check_attention((q, kp, vp, table, cu, lens), 0.25, causal)
    for clip in (130, 900):  # keys before these have the lowest of all, and the first rows see no others
        kp[table[0, at // 16].long(), 0, at % 16, 0] = torch.where(at < clip, -(2.0**66), 0.0).to(torch.bfloat16)
        _check_attention((q, kp, vp, table, cu, lens), 0.25, causal)


def test_results_of_the_registered_plans_share_no_memory():
    """As their schemas say; the direct call's are pieces of one allocation, apart from the state in place."""
    from tybok_b200 import ops

    state = lambda: (_i32([16, 4]), _i32([1, 2]), torch.zeros(2, 5000, dtype=torch.int32, device="cuda"), _i32([2, 3, 0]), _i32([2]))  # noqa: E731
    where = lambda t: t.untyped_storage().data_ptr()  # noqa: E731
    plan, own = ops.page_plan(*state(), tokens=3, page_size=16), ops.page_plan_(*state(), tokens=3, page_size=16)
    for t in (own.cu_tokens, own.pos, own.slots, own.missing):
        assert where(t) != where(own.block_table) and t.untyped_storage().nbytes() < 4096
    for out in (torch.ops.tybok_b200.page_plan(*state(), 3, 16, None), torch.ops.tybok_b200.page_plan_(*state(), 3, 16, None)):
        assert len({where(t) for t in out}) == len(out)
        assert all(torch.equal(a, b) for a, b in zip(out, plan if len(out) == 8 else plan[4:]))


@pytest.mark.parametrize("h,g,d,most", [(8, 1, 256, 240), (8, 2, 128, 240), (1, 1, 128, 1), (8, 1, 256, 1)])
@pytest.mark.parametrize("cu,lens", [([0, 240, 0, 240, 0, 240, 0], [60] * 6), ([0, -5, 300, 240, 1 << 30, -(1 << 31), 7], [60, 1 << 30, -1, 0, 500, 3]),
                                     ([230, 240, 250, 260, 0, 10, 500], [400] * 6)])
def test_bounds_out_of_range_touch_no_byte_around_the_outputs(h, g, d, most, cu, lens):
    """Through the C entry point, with outputs, planes and workspace inside larger tensors of a pattern."""
    import ctypes

    from tybok_b200 import _lib, ops

    q, kp, vp, table, _, _ = _attention_inputs([60] * 6, [40] * 6, h, g, d, 16, seed=12)
    lib, n, edge = _lib.load(), q.numel(), 1 << 20
    need = lib.tybok_paged_attention_workspace_bytes(h, g, d, most)
    whole = {"out": torch.full((2 * n + 2 * edge,), 0x5A, dtype=torch.uint8, device="cuda"),
             "planes": torch.full((3 * n + 2 * edge,), 0x5A, dtype=torch.uint8, device="cuda"),
             "ws": torch.full((need + 2 * edge,), 0x5A, dtype=torch.uint8, device="cuda")}
    strides = lambda t: (ctypes.c_int64 * 3)(*t.stride()[:3])  # noqa: E731
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    cu_t, lens_t = _i32(cu), _i32(lens)
    at = {name: t.data_ptr() + edge for name, t in whole.items()}
    rc = lib.tybok_paged_attention(q.data_ptr(), q.stride(0), kp.data_ptr(), strides(kp), vp.data_ptr(), strides(vp), table.data_ptr(), table.stride(0),
                                   cu_t.data_ptr(), lens_t.data_ptr(), at["out"], at["planes"], 3, q.shape[0], 6, h, g, d, kp.shape[0], 16, table.shape[1],
                                   most, 0, 0.08, at["ws"], need, word.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.tybok_last_error()
    assert word.item() == ops.DEV_BAD_INDEX
    for name, t in whole.items():
        assert bool((t[:edge] == 0x5A).all()) and bool((t[-edge:] == 0x5A).all()), name
