"""What the paged cache's operators refuse before they launch anything (the checks come before the test for a CUDA tensor: a call
whose sizes agree ends in ``NotImplementedError``), and the C entry points' own checks."""

import ctypes

import pytest
import torch

B, W, P, PAGE, T, H, G, D = 3, 4, 20, 16, 9, 4, 2, 128


def _i(*shape, fill=0):
    return torch.full(shape, fill, dtype=torch.int32)


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def _plan(in_place=False, **over):
    from tybok_b200 import ops

    args = dict(key_lens=_i(B), new_lens=_i(B, fill=1), block_table=_i(B, W), free_pages=_i(P), free_count=_i(1, fill=P))
    kw = dict(tokens=T, page_size=PAGE, finished=None)
    args.update({k: v for k, v in over.items() if k in args})
    kw.update({k: v for k, v in over.items() if k in kw})
    return (ops.page_plan_ if in_place else ops.page_plan)(*args.values(), **kw)


def _store(**over):
    from tybok_b200 import ops

    args = dict(qkv=_bf(T, (H + 2 * G) * D), pos=_i(T), slots=_i(T), cos=torch.zeros(64, D // 2), sin=torch.zeros(64, D // 2),
                k_pages=_bf(P, G, PAGE, D), v_pages=_bf(P, G, PAGE, D))
    kw = dict(heads=H, norm_q=torch.ones(D), norm_k=torch.ones(D), eps=1e-6, paired=False)
    args.update({k: v for k, v in over.items() if k in args})
    kw.update({k: v for k, v in over.items() if k in kw})
    return ops.head_norm_rope_store(*args.values(), **kw)


def _attend(**over):
    from tybok_b200 import ops

    args = dict(q=_bf(T, H * D), k_pages=_bf(P, G, PAGE, D), v_pages=_bf(P, G, PAGE, D), block_table=_i(B, W), cu_tokens=_i(B + 1),
                key_lens=_i(B))
    kw = dict(scale=0.1, causal=True, max_tokens=None, out_bf16=True, out_planes=False, out_shift=4)
    args.update({k: v for k, v in over.items() if k in args})
    kw.update({k: v for k, v in over.items() if k in kw})
    return ops.paged_attention(*args.values(), **kw)


@pytest.mark.parametrize("call", [
    lambda: _plan(), lambda: _plan(True), lambda: _plan(finished=torch.zeros(B, dtype=torch.bool)),
    lambda: _plan(finished=torch.zeros(B, dtype=torch.uint8)), lambda: _store(), lambda: _store(norm_q=None, norm_k=None),
    lambda: _store(cos=torch.zeros(64, 24), sin=torch.zeros(64, 24)), lambda: _store(k_pages=_bf(P, PAGE, G, D).transpose(1, 2)),
    lambda: _store(qkv=_bf(T, (H + 2 * G) * D + 1)[:, 1:]),  # copied
    lambda: _attend(), lambda: _attend(max_tokens=1), lambda: _attend(out_planes=True), lambda: _attend(block_table=_i(B, W + 3)[:, :W]),
    lambda: _attend(k_pages=_bf(P, 2, G, PAGE, D)[:, 0]),
])
def test_agreeing_calls_only_lack_a_gpu(call):
    with pytest.raises(NotImplementedError, match="no CPU implementation|'CPU' backend"):
        call()


@pytest.mark.parametrize("over", [
    dict(key_lens=_i(B).long()), dict(new_lens=_i(B + 1)), dict(new_lens=torch.ones(B)), dict(block_table=_i(B + 1, W)),
    dict(block_table=_i(W, B).t()), dict(block_table=_i(B, 0)), dict(block_table=_i(B, W).long()), dict(free_pages=_i(2 * P)[::2]),
    dict(free_pages=_i(0)), dict(free_count=_i(2)), dict(finished=_i(B)), dict(finished=torch.zeros(B - 1, dtype=torch.bool)),
    dict(tokens=-1), dict(page_size=0), dict(key_lens=_i(0), new_lens=_i(0), block_table=_i(0, W)),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_refuses(over, in_place):
    with pytest.raises((TypeError, ValueError)):
        _plan(in_place, **over)


@pytest.mark.parametrize("over", [
    dict(qkv=_bf(T, (H + 2 * G) * D - 8)), dict(qkv=torch.zeros(T, (H + 2 * G) * D)), dict(heads=H + 1), dict(heads=0), dict(pos=_i(T - 1)),
    dict(pos=_i(T).long()), dict(slots=_i(T + 1)), dict(slots=_i(2 * T)[::2]), dict(cos=torch.zeros(64, D // 2).double()),
    dict(sin=torch.zeros(63, D // 2)), dict(cos=torch.zeros(D // 2, 64).t(), sin=torch.zeros(D // 2, 64).t()),
    dict(k_pages=_bf(P, G, PAGE, D).half()), dict(v_pages=_bf(P, G, PAGE + 16, D)), dict(k_pages=_bf(G, PAGE, D)),
    dict(k_pages=_bf(P, G, D, PAGE).transpose(2, 3), v_pages=_bf(P, G, D, PAGE).transpose(2, 3)),
    dict(k_pages=_bf(1, G, PAGE, D).expand(P, G, PAGE, D)),  # pages on top of one another
    dict(k_pages=_bf(P * G * PAGE * D + 8)[4:-4].view(P, G, PAGE, D)),  # not aligned
    dict(norm_q=torch.ones(D - 1)), dict(norm_k=_bf(D)), dict(cos=torch.zeros(64, D + 8), sin=torch.zeros(64, D + 8)),
])
def test_store_refuses(over):
    with pytest.raises((TypeError, ValueError)):
        _store(**over)


@pytest.mark.parametrize("over", [
    dict(q=_bf(T, 3 * D)), dict(q=_bf(T, H * D + 8)), dict(q=torch.zeros(T, H * D)), dict(q=_bf(1, T, H * D)), dict(q=_bf(T, 0)),
    dict(k_pages=_bf(P, G, PAGE, D).float()), dict(v_pages=_bf(P + 1, G, PAGE, D)), dict(block_table=_i(B - 1, W)),
    dict(block_table=_i(W, B).t()), dict(block_table=_i(B, W).long()), dict(cu_tokens=_i(B)), dict(cu_tokens=_i(B + 1).long()),
    dict(key_lens=_i(B + 1)), dict(key_lens=_i(0), cu_tokens=_i(1), block_table=_i(0, W)), dict(max_tokens=0), dict(out_bf16=False),
    dict(k_pages=_bf(1, G, PAGE, D).expand(P, G, PAGE, D)), dict(v_pages=_bf(P, 1, PAGE, D).expand(P, G, PAGE, D)),
])
def test_attention_refuses(over):
    with pytest.raises((TypeError, ValueError)):
        _attend(**over)


def _c(entry, **over):
    """A C call whose arguments agree, but for `over`; stops at the checks (16 stands for a pointer that nobody follows)."""
    from tybok_b200 import _lib

    ptr, strides = ctypes.c_void_p(16), (ctypes.c_int64 * 3)(G * PAGE * D, PAGE * D, D)
    if entry == "tybok_page_plan":
        args = {f"p{i}": ptr for i in range(6)}
        args.update({f"o{i}": ctypes.c_void_p(32) for i in range(8)}, B=B, width=W, pages=P, tokens=T, page=PAGE, stream=None)
    elif entry == "tybok_head_norm_rope_store":
        args = dict(src=ptr, ld=(H + 2 * G) * D, pos=ptr, slots=ptr, cos=ptr, sin=ptr, max_pos=64, rot=D, paired=0, nq=ptr, nk=ptr, eps=1e-6,
                    q=ptr, k=ptr, ks=strides, v=ptr, vs=strides, tokens=T, H=H, G=G, D=D, pages=P, page=PAGE, status=None, stream=None)
    else:
        args = dict(q=ptr, ldq=H * D, k=ptr, ks=strides, v=ptr, vs=strides, table=ptr, ldt=W, cu=ptr, lens=ptr, out=ptr, planes=None, shift=4,
                    tokens=T, B=B, H=H, G=G, D=D, pages=P, page=PAGE, width=W, most=T, causal=1, scale=0.1, ws=ptr, bytes=1 << 40, status=None,
                    stream=None)
    args.update(over)
    lib = _lib.load()
    return getattr(lib, entry)(*args.values()), lib.tybok_last_error().decode()


@pytest.mark.parametrize("entry,over,says", [
    ("tybok_page_plan", dict(p0=None), "null"), ("tybok_page_plan", dict(page=24), "power of two"), ("tybok_page_plan", dict(page=8), "power of two"),
    ("tybok_page_plan", dict(B=0), "bad shape"), ("tybok_page_plan", dict(B=8193), "bad shape"), ("tybok_page_plan", dict(pages=1 << 28), "31 bits"),
    ("tybok_page_plan", dict(o0=ctypes.c_void_p(16)), "in place"),
    ("tybok_head_norm_rope_store", dict(q=None), "null"), ("tybok_head_norm_rope_store", dict(D=64), "head_dim"),
    ("tybok_head_norm_rope_store", dict(rot=24), "bad shape"), ("tybok_head_norm_rope_store", dict(rot=D + 16), "bad shape"),
    ("tybok_head_norm_rope_store", dict(rot=0), "bad shape"), ("tybok_head_norm_rope_store", dict(tokens=0), "bad shape"),
    ("tybok_head_norm_rope_store", dict(page=17), "power of two"), ("tybok_head_norm_rope_store", dict(ld=(H + 2 * G) * D + 4), "aligned"),
    ("tybok_head_norm_rope_store", dict(k=ctypes.c_void_p(8)), "aligned"), ("tybok_head_norm_rope_store", dict(pages=1 << 28), "31 bits"),
    ("tybok_paged_attention", dict(q=None), "null"), ("tybok_paged_attention", dict(out=None), "null"),
    ("tybok_paged_attention", dict(D=64), "head_dim"), ("tybok_paged_attention", dict(H=3), "bad shape"),
    ("tybok_paged_attention", dict(B=2049), "bad shape"), ("tybok_paged_attention", dict(page=48), "power of two"),
    ("tybok_paged_attention", dict(ldq=H * D + 4), "aligned"), ("tybok_paged_attention", dict(v=ctypes.c_void_p(24)), "aligned"),
    ("tybok_paged_attention", dict(shift=61), "exponent"), ("tybok_paged_attention", dict(ws=None), "workspace"),
    ("tybok_paged_attention", dict(bytes=16), "workspace"), ("tybok_paged_attention", dict(tokens=1 << 30), "31 bits"),
    ("tybok_paged_attention", dict(width=1 << 27), "31 bits"), ("tybok_paged_attention", dict(ks=(ctypes.c_int64 * 3)(0, PAGE * D, D)), "positive"),
    ("tybok_head_norm_rope_store", dict(vs=(ctypes.c_int64 * 3)(G * PAGE * D, 0, D)), "positive"),
])
def test_c_entry_points_refuse(entry, over, says):
    rc, message = _c(entry, **over)
    assert rc != 0 and says in message


def test_workspace_is_bounded():
    from tybok_b200 import _lib

    lib = _lib.load()
    for h, g, d, n in ((8, 1, 256, 1), (8, 1, 256, 50), (32, 8, 128, 4096), (1, 1, 128, 1 << 20)):
        assert 0 < lib.tybok_paged_attention_workspace_bytes(h, g, d, n) <= 100 << 20
    assert lib.tybok_paged_attention_workspace_bytes(8, 1, 64, 1) == 0


SAME = _bf(P, G, PAGE, D)


@pytest.mark.parametrize("over", [
    dict(k_pages=SAME, v_pages=SAME),
    dict(k_pages=_bf(P * G * PAGE * D).as_strided((P, G, PAGE, D), (G * PAGE * D, PAGE * D, D // 2, 1))),  # rows half on one another
    dict(v_pages=_bf(P * G * PAGE * D).as_strided((P, G, PAGE, D), (PAGE * D, PAGE * D, D, 1))),  # heads in the next page
    dict(v_pages=_bf(P * G * PAGE * D).as_strided((P, G, PAGE, D), (8, PAGE * D, D, 1))),
])
def test_store_refuses_rows_on_top_of_one_another(over):
    with pytest.raises(ValueError, match="overlap"):
        _store(**over)


@pytest.mark.parametrize("shape,strides", [
    ((P, G, PAGE, D), (D, P * D, P * G * D, 1)), ((P, 1, PAGE, D), (PAGE * D, 8, D, 1)), ((1, G, PAGE, D), (8, D, G * D, 1)),
    ((P, G, PAGE, D), (2 * G * PAGE * (D + 8), PAGE * (D + 8), D + 8, 1)),
])
def test_store_takes_any_order_of_rows_that_lie_apart(shape, strides):
    pool = lambda: _bf(4 * P * G * PAGE * D).as_strided(shape, strides)  # noqa: E731
    heads = H + 2 * G - 2 * shape[1]
    with pytest.raises(NotImplementedError, match="no CPU implementation|'CPU' backend"):
        _store(k_pages=pool(), v_pages=pool(), heads=heads)


@pytest.mark.parametrize("over", [
    dict(v=ctypes.c_void_p(16)), dict(ks=(ctypes.c_int64 * 3)(G * PAGE * D, PAGE * D, D - 8)), dict(vs=(ctypes.c_int64 * 3)(PAGE * D, PAGE * D, D)),
    dict(ks=(ctypes.c_int64 * 3)(1 << 62, 1 << 62, D)),
])
def test_c_store_refuses_rows_on_top_of_one_another(over):
    rc, message = _c("tybok_head_norm_rope_store", **{"v": ctypes.c_void_p(32), **over})
    assert rc != 0 and "overlap" in message
