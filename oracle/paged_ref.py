"""The paged cache's operators in plain form: the page plan request by request on the host, the floating ones in 64 bits."""

from __future__ import annotations

import math

import torch


def pages(n: int, page: int) -> int:
    return -(-n // page)


def page_plan(key_lens, new_lens, block_table, free_pages, free_count, *, tokens, page_size, finished=None):
    """``(key_lens, block_table, free_pages, free_count, cu_tokens, pos, slots, missing)`` as lists."""
    lens, new, table, stack, count = (t.tolist() for t in (key_lens, new_lens, block_table, free_pages, free_count))
    gone = [False] * len(lens) if finished is None else [bool(x) for x in finished.tolist()]
    width, count = len(table[0]), count[0]
    base = [0 if out else n for n, out in zip(lens, gone)]
    back = [pages(n, page_size) if out else 0 for n, out in zip(lens, gone)]
    more = [pages(b + n, page_size) - pages(b, page_size) for b, n in zip(base, new)]
    bad = any(n < 0 for n in lens + new) or any(pages(n, page_size) > width for n in lens) or any(
        pages(b + n, page_size) > width for b, n in zip(base, new)) or sum(new) > tokens or not 0 <= count <= len(stack) \
        or count + sum(back) > len(stack)
    missing = -1 if bad else max(0, sum(more) - count - sum(back))
    if missing:
        return lens, table, stack, [count], [0] * (len(lens) + 1), [0] * tokens, [-1] * tokens, [missing]
    for b, n in enumerate(back):
        stack[count : count + n] = table[b][:n]
        count += n
    pos, slots, cu = [], [], [0]
    for b, n in enumerate(new):
        for j in range(pages(base[b], page_size), pages(base[b] + n, page_size)):
            count -= 1
            table[b][j] = stack[count]
        for p in range(base[b], base[b] + n):
            pos.append(p)
            slots.append(table[b][p // page_size] * page_size + p % page_size)
        cu.append(cu[-1] + n)
    behind = tokens - len(pos)
    return [b + n for b, n in zip(base, new)], table, stack, [count], cu, pos + [0] * behind, slots + [-1] * behind, [0]


def head_norm_rope(x, pos, cos, sin, weight, eps, paired):
    """``x [T, heads, D]`` -> (result, sum of the magnitudes of its two terms), float64."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    r = 2 * cos.shape[1]
    c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
    y, size = x.clone(), x.abs()
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if paired else (x[..., : r // 2], x[..., r // 2 : r])
    ya, yb = a * c - b * s, b * c + a * s
    na, nb = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    if paired:
        y[..., 0:r:2], y[..., 1:r:2], size[..., 0:r:2], size[..., 1:r:2] = ya, yb, na, nb
    else:
        y[..., : r // 2], y[..., r // 2 : r], size[..., : r // 2], size[..., r // 2 : r] = ya, yb, na, nb
    return y, size


def paged_attention(q, k_pages, v_pages, block_table, cu_tokens, key_lens, *, scale, causal):
    """-> (output ``[T, H*D]``, the same average of the values' magnitudes), float64; rows of no request and queries that see no
    key are zero."""
    _, g, page, d = k_pages.shape
    h = q.shape[1] // d
    out, size = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    cu, lens = cu_tokens.tolist(), key_lens.tolist()
    for b, n_keys in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0 or n_keys == 0:
            continue
        at = torch.arange(n_keys, device=q.device)
        where, row = block_table[b].long()[at // page], at % page
        seen = torch.ones(n, n_keys, dtype=torch.bool, device=q.device)
        if causal:
            seen = at[None] <= (n_keys - n + torch.arange(n, device=q.device))[:, None]
        for head in range(h):
            k, v = k_pages[where, head // (h // g), row].double(), v_pages[where, head // (h // g), row].double()
            s = (q[cu[b] : cu[b + 1], head * d : (head + 1) * d].double() @ k.T) * scale
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True)
            e = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            w = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
            out[cu[b] : cu[b + 1], head * d : (head + 1) * d] = w @ v
            size[cu[b] : cu[b + 1], head * d : (head + 1) * d] = w @ v.abs()
    return out, size
