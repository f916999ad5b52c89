"""What the paged cache of keys and values is measured on: its three operators, each as one call of a user's program.

``plan``   ``ops.page_plan``: pages, block tables, positions and slots of a step from the requests' lengths.
``store``  ``ops.head_norm_rope_store``: norms of queries and keys for each head, rotation, keys and values into their pages.
``attend`` ``ops.paged_attention``: new tokens over the pages of their requests.

Every case has the plain form of its operator beside it (elementary torch operations in 32 bits, whole numbers in 64) and
the definition in 64 bits (``exact``).
"""

from __future__ import annotations

import math
import random

import torch

DEVICE = "cuda"
own = False


def listed() -> list[dict]:
    return [
        # A step of a small fleet: every request brings one token, a few leave and their rows are taken over.
        plan_case("plan_step_48", batch=48, page=16, past=(1, 2000), new=(1, 1), leave=0.06, lens=1),
        # Prompts of very different lengths enter beside requests that wait (no new token).
        plan_case("plan_prompts_7", batch=7, page=64, past=(0, 700), new=(0, 1500), leave=0.2, lens=2),
        # A large pool: two thousand requests, most of them in their prompts, small pages.
        plan_case("plan_pool_2048", batch=2048, page=16, past=(0, 1500), new=(1, 90), leave=0.1, lens=3),
        # One layer of a step of 33 single tokens at the policy decoders' heads.
        store_case("store_step_33", tokens=33, heads=8, kv_heads=1, head_dim=256, page=16, paired=False, spare=7),
        # A ragged chunk at as many key heads as query heads, rotated pair-wise.
        store_case("store_chunk_777", tokens=777, heads=16, kv_heads=16, head_dim=128, page=64, paired=True, spare=23),
        # Prompts of a whole batch, grouped heads: memory traffic beyond the second-level cache.
        store_case("store_prompts_16384", tokens=16384, heads=32, kv_heads=8, head_dim=128, page=32, paired=False, spare=0),
        # Three requests, one token each, short caches: the smallest call, latency counts.
        attend_case("attend_step_3", batch=3, heads=8, kv_heads=1, head_dim=256, page=16, past=(1, 600), new=(1, 1), causal=True,
                    lens=4),
        # Single tokens over long caches of very different lengths: the rate of memory.
        attend_case("attend_step_64", batch=64, heads=32, kv_heads=8, head_dim=128, page=32, past=(500, 16000), new=(1, 1),
                    causal=True, lens=5),
        # The action chunk of eight robots over prefixes of one to three cameras: all keys are visible to all queries.
        attend_case("attend_suffix_8", batch=8, heads=8, kv_heads=1, head_dim=256, page=64, past=(258, 968), new=(50, 50),
                    causal=False, lens=6),
        # The prefixes themselves, of odd lengths, with nothing in the cache before.
        attend_case("attend_prefix_5", batch=5, heads=8, kv_heads=1, head_dim=256, page=16, past=(0, 0), new=(401, 968), causal=False,
                    lens=7),
        # A step that mixes single tokens with pieces of prompts.
        attend_case("attend_mixed_19", batch=19, heads=16, kv_heads=16, head_dim=128, page=16, past=(3, 5000), new=(1, 700),
                    causal=True, lens=8),
        # Large pieces of long prompts: matrix products.
        attend_case("attend_chunk_2048", batch=2, heads=32, kv_heads=8, head_dim=128, page=128, past=(6000, 6500), new=(2048, 2048),
                    causal=True, lens=9),
    ]


def plan_case(name, *, batch, page, past, new, leave, lens):
    return {"name": name, "op": "plan", "batch": batch, "page": page, "past_lo": past[0], "past_hi": past[1], "new_lo": new[0],
            "new_hi": new[1], "leave": leave, "lens": lens}


def store_case(name, *, tokens, heads, kv_heads, head_dim, page, paired, spare):
    return {"name": name, "op": "store", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "paired": paired, "spare": spare}


def attend_case(name, *, batch, heads, kv_heads, head_dim, page, past, new, causal, lens):
    return {"name": name, "op": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "past_lo": past[0], "past_hi": past[1], "new_lo": new[0], "new_hi": new[1], "causal": causal, "lens": lens}


# Heads of the policy decoders, of the denoiser's kind (as many key heads as query heads), and grouped ones.
HEADS = ((8, 1, 256), (16, 16, 128), (32, 8, 128), (12, 4, 128), (16, 2, 128), (2, 1, 128), (6, 2, 256), (10, 2, 128))


def _spread(rng, lo, hi):
    """A whole number between the two, spread over its logarithm (zero stands one below one)."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))) - 1)))


def draw(rng: random.Random) -> dict:
    op = rng.choice(("plan", "store", "attend", "attend"))
    page = rng.choice((16, 32, 64, 128))
    if op == "plan":
        batch = _spread(rng, 1, 2048)
        hi = _spread(rng, 1, max(1, min(4000, 90000 // batch)))
        past = min(_spread(rng, 0, 16000), 3000000 // batch)
        case = plan_case("", batch=batch, page=page, past=(0, past), new=(rng.choice((0, 1)), hi), leave=rng.choice((0.0, 0.1, 0.5)),
                         lens=rng.randrange(1 << 30))
    elif op == "store":
        heads, kv, dim = rng.choice(HEADS)
        case = store_case("", tokens=_spread(rng, 1, 16384 * 48 * 128 // ((heads + 2 * kv) * dim)), heads=heads, kv_heads=kv, head_dim=dim,
                          page=page, paired=rng.random() < 0.5, spare=rng.choice((0, 1, 30)))
    else:
        heads, kv, dim = rng.choice(HEADS)
        batch = _spread(rng, 1, 64)
        single = rng.random() < 0.4
        new = 1 if single else _spread(rng, 2, min(2048, 4096 // batch))
        past = _spread(rng, 0, min(16000, 500000 // batch))
        while batch * new * (past + new) * heads * dim > 2 * 2048 * 7000 * 32 * 128 or batch * (past + new) * kv * dim > 64 * 8000 * 8 * 128:
            past, new = past // 2, (new + 1) // 2
        case = attend_case("", batch=batch, heads=heads, kv_heads=kv, head_dim=dim, page=page, past=(past // 4, past),
                           new=(1, new) if rng.random() < 0.5 else (new, new), causal=rng.random() < 0.7, lens=rng.randrange(1 << 30))
    del case["name"]
    return case


def lengths(case: dict) -> tuple[list[int], list[int]]:
    """Keys each request holds before the step and new tokens it brings: part of the case, not of the seed."""
    rng = random.Random(case["lens"])
    past = [_spread(rng, case["past_lo"], case["past_hi"]) for _ in range(case["batch"])]
    new = [_spread(rng, case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    return past, new


def leaving(case: dict) -> list[bool]:
    rng = random.Random(case["lens"] + 1)
    return [rng.random() < case["leave"] for _ in range(case["batch"])]


def _pages(n: int, page: int) -> int:
    return -(-n // page)


def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


# ---------------------------------------------------------------------------------------------------------------- inputs
def prepare(case: dict, seed: int) -> dict:
    return {"plan": _prepare_plan, "store": _prepare_store, "attend": _prepare_attend}[case["op"]](case, seed)


def _prepare_plan(case, seed):
    past, new = lengths(case)
    page, b = case["page"], case["batch"]
    width = max(_pages(p + n, page) for p, n in zip(past, new)) + 3
    held = [_pages(p, page) for p in past]
    total = sum(held) + sum(_pages(p + n, page) for p, n in zip(past, new)) + 5
    pages = torch.randperm(total, generator=_generator(seed), device=DEVICE).to(torch.int32)
    table = torch.zeros(b, width, dtype=torch.int32, device=DEVICE)
    col = torch.arange(width, device=DEVICE)[None]
    mask = col < torch.tensor(held, device=DEVICE)[:, None]
    n_held = sum(held)
    table[mask] = pages[:n_held]
    free = torch.zeros(total, dtype=torch.int32, device=DEVICE)
    free[: total - n_held] = pages[n_held:]
    tokens = sum(new) + 5
    return {"case": case, "key_lens": _ints(past), "new_lens": _ints(new), "finished": torch.tensor(leaving(case), device=DEVICE),
            "table": table, "free": free, "count": _ints([total - n_held]), "tokens": tokens}


def _prepare_store(case, seed):
    gen = _generator(seed)
    t, h, g, d, page = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    rows = t + case["spare"]
    qkv = torch.randn(rows, (h + 2 * g) * d, generator=gen, device=DEVICE).to(torch.bfloat16)
    n_pages = _pages(t, page) + 2
    # pages in any order, the first one begun by earlier tokens; rows behind the last token have no slot
    order = torch.randperm(n_pages, generator=gen, device=DEVICE)
    first = page // 3
    at = torch.arange(t, device=DEVICE) + first
    slots = torch.full((rows,), -1, dtype=torch.int32, device=DEVICE)
    slots[:t] = (order[at // page] * page + at % page).to(torch.int32)
    pos = torch.zeros(rows, dtype=torch.int32, device=DEVICE)
    pos[:t] = (at % 4001).to(torch.int32)
    angle = torch.arange(4096, dtype=torch.float64, device=DEVICE)[:, None] * (
        10000.0 ** (-torch.arange(d // 2, dtype=torch.float64, device=DEVICE) / (d // 2)))[None]
    cache = lambda: torch.randn(n_pages, g, page, d, generator=gen, device=DEVICE).to(torch.bfloat16)  # noqa: E731
    weight = lambda: 1.0 + 0.2 * torch.randn(d, generator=gen, device=DEVICE)  # noqa: E731
    return {"case": case, "qkv": qkv, "pos": pos, "slots": slots, "cos": angle.cos().float(), "sin": angle.sin().float(),
            "norm_q": weight(), "norm_k": weight(), "k_pages": cache(), "v_pages": cache()}


def _prepare_attend(case, seed):
    gen = _generator(seed)
    past, new = lengths(case)
    h, g, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    totals = [p + n for p, n in zip(past, new)]
    n_pages = sum(_pages(x, page) for x in totals) + 3
    order = torch.randperm(n_pages, generator=gen, device=DEVICE).to(torch.int32)
    width = max(_pages(x, page) for x in totals) + 1
    table = torch.zeros(case["batch"], width, dtype=torch.int32, device=DEVICE)
    mask = torch.arange(width, device=DEVICE)[None] < torch.tensor([_pages(x, page) for x in totals], device=DEVICE)[:, None]
    table[mask] = order[: int(sum(_pages(x, page) for x in totals))]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = torch.randn(starts[-1], h * d, generator=gen, device=DEVICE).to(torch.bfloat16)
    cache = lambda: torch.randn(n_pages, g, page, d, generator=gen, dtype=torch.bfloat16, device=DEVICE)  # noqa: E731
    return {"case": case, "q": q, "k_pages": cache(), "v_pages": cache(), "table": table, "cu_tokens": _ints(starts),
            "key_lens": _ints(totals), "max_tokens": max(new)}


# ----------------------------------------------------------------------------------------------------------------- calls
def run(state: dict):
    case = state["case"]
    if not own:
        return {"plan": _plain_plan, "store": _plain_store, "attend": _plain_attend}[case["op"]](state)
    from tybok_b200 import ops

    s = state
    if case["op"] == "plan":
        plan = ops.page_plan(s["key_lens"], s["new_lens"], s["table"], s["free"], s["count"], tokens=s["tokens"], page_size=case["page"],
                             finished=s["finished"])
        return [plan.key_lens, plan.block_table, plan.free_pages, plan.free_count, plan.cu_tokens, plan.pos, plan.slots, plan.missing]
    if case["op"] == "store":
        q = ops.head_norm_rope_store(s["qkv"], s["pos"], s["slots"], s["cos"], s["sin"], s["k_pages"], s["v_pages"], heads=case["heads"],
                                     norm_q=s["norm_q"], norm_k=s["norm_k"], eps=1e-6, paired=case["paired"])
        return [q, s["k_pages"], s["v_pages"]]
    out, _ = ops.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cu_tokens"], s["key_lens"], scale=case["head_dim"] ** -0.5,
                                 causal=case["causal"], max_tokens=s["max_tokens"])
    return [out]


def _plain_plan(s):
    page, rows = s["case"]["page"], s["tokens"]
    lens, new, table, free, count = s["key_lens"].long(), s["new_lens"].long(), s["table"].long(), s["free"].long(), s["count"].long()
    width, n_pages = table.shape[1], free.shape[0]
    out = s["finished"]
    held = (lens + page - 1) // page
    base = torch.where(out, torch.zeros_like(lens), lens)
    keep = torch.where(out, torch.zeros_like(held), held)
    total = base + new
    need = (total + page - 1) // page
    back, more = held - keep, need - keep
    n_back, n_more = back.sum(), more.sum()
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=lens.device), new.cumsum(0)])
    short = (n_more - count[0] - n_back).clamp(min=0)
    bad = (lens < 0).any() | (new < 0).any() | (cu[-1] > rows) | (torch.maximum(held, need) > width).any() | (count[0] + n_back > n_pages)
    missing = torch.where(bad, torch.full_like(short, -1), short)
    ok = missing == 0
    col = torch.arange(width, device=lens.device)[None]
    # pages that come back, on top of the stack
    stack = torch.cat([free, free.new_zeros(1)])  # the last entry takes what has no place
    at = count[0] + (back.cumsum(0) - back)[:, None] + col
    stack[torch.where((col < back[:, None]) & ok, at, n_pages)] = table
    # pages that are taken, from its top
    which = (more.cumsum(0) - more)[:, None] + col - keep[:, None]
    taken = stack[(count[0] + n_back - 1 - which).clamp(0, n_pages - 1)]
    table = torch.where((col >= keep[:, None]) & (col < need[:, None]) & ok, taken, table)
    token = torch.arange(rows, device=lens.device)
    row = torch.searchsorted(cu[1:].contiguous(), token, right=True).clamp(max=lens.shape[0] - 1)
    real = (token < cu[-1]) & ok
    pos = torch.where(real, base[row] + token - cu[row], 0)
    slots = torch.where(real, table[row, (pos // page).clamp(max=width - 1)] * page + pos % page, -1)
    i32 = lambda t: t.to(torch.int32)  # noqa: E731
    return [i32(torch.where(ok, total, lens)), i32(table), i32(stack[:n_pages]), i32(torch.where(ok, count + n_back - n_more, count)),
            i32(torch.where(ok, cu, torch.zeros_like(cu))), i32(pos), i32(slots), i32(missing.reshape(1))]


def _plain_store(s):
    case = s["case"]
    h, g, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    x = s["qkv"].view(-1, h + 2 * g, d).float()
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]

    def turned(x, weight):
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
        if case["paired"]:
            a, b = x[..., 0::2], x[..., 1::2]
            return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
        a, b = x[..., : d // 2], x[..., d // 2 :]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)

    q = turned(x[:, :h], s["norm_q"]).to(torch.bfloat16)
    k = turned(x[:, h : h + g], s["norm_k"]).to(torch.bfloat16)
    t = case["tokens"]  # rows behind them have no slot
    slots = s["slots"][:t].long()
    s["k_pages"][slots // page, :, slots % page] = k[:t]
    s["v_pages"][slots // page, :, slots % page] = s["qkv"].view(-1, h + 2 * g, d)[:t, h + g :]
    return [q.reshape(-1, h * d), s["k_pages"], s["v_pages"]]


def _plain_attend(s):
    case = s["case"]
    h, g, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    past, new = lengths(case)
    out = torch.zeros_like(s["q"])
    at = 0
    for b, (p, n) in enumerate(zip(past, new)):
        keys = p + n
        rows = s["table"][b, : _pages(keys, page)].long()
        k, v = (c[rows].transpose(0, 1).reshape(g, -1, d)[:, :keys].float() for c in (s["k_pages"], s["v_pages"]))
        q = s["q"][at : at + n].view(n, g, h // g, d).permute(1, 2, 0, 3).float()  # [G, H/G, n, D]
        score = (q @ k[:, None].transpose(-1, -2)) * d**-0.5
        if case["causal"] and n > 1:
            seen = torch.arange(keys, device=q.device)[None] <= p + torch.arange(n, device=q.device)[:, None]
            score = score.masked_fill(~seen, -math.inf)
        e = torch.exp(score - score.amax(-1, keepdim=True))
        y = (e @ v[:, None]) / e.sum(-1, keepdim=True)
        out[at : at + n] = y.permute(2, 0, 1, 3).reshape(n, h * d).to(torch.bfloat16)
        at += n
    return [out]


# ------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case: dict) -> dict:
    if case["op"] == "store":
        row = (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        return {"bytes": 2 * 2 * row * case["tokens"] + 8 * case["tokens"] + 4 * case["head_dim"] * min(case["tokens"], 4001),
                "flops": 7 * row * case["tokens"]}
    past, new = lengths(case)
    page, b = case["page"], case["batch"]
    if case["op"] == "plan":
        out = leaving(case)
        back = sum(_pages(p, page) for p, o in zip(past, out) if o)
        more = sum(_pages((0 if o else p) + n, page) - (0 if o else _pages(p, page)) for p, n, o in zip(past, new, out))
        width = max(_pages(p + n, page) for p, n in zip(past, new)) + 3
        stack = sum(_pages(p, page) + _pages(p + n, page) for p, n in zip(past, new)) + 5
        # lengths and flags, the table and the stack in and out, positions and slots out
        return {"bytes": 9 * b + 8 * b * width + 8 * stack + 4 * (2 * b + 1) + 8 * (sum(new) + 5) + 8, "flops": 8 * sum(new) + 4 * (back + more)}
    h, g, d = case["heads"], case["kv_heads"], case["head_dim"]
    pairs = sum(n * p + (n * (n + 1) // 2 if case["causal"] else n * n) for p, n in zip(past, new))
    keys = sum(p + n for p, n in zip(past, new))
    return {"bytes": 2 * 2 * sum(new) * h * d + 2 * 2 * keys * g * d + 4 * sum(_pages(p + n, page) for p, n in zip(past, new)) + 8 * b + 4,
            "flops": 4 * h * d * pairs}


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "store": _exact_store, "attend": _exact_attend}[case["op"]](s)


def _exact_plan(s):
    """Request by request, on the host."""
    page = s["case"]["page"]
    lens, new, out = s["key_lens"].tolist(), s["new_lens"].tolist(), s["finished"].tolist()
    table, free, count = s["table"].tolist(), s["free"].tolist(), s["count"].tolist()[0]
    for b, gone in enumerate(out):
        if gone:
            for j in range(_pages(lens[b], page)):
                free[count] = table[b][j]
                count += 1
            lens[b] = 0
    pos, slots, cu = [], [], [0]
    for b, n in enumerate(new):
        for j in range(_pages(lens[b], page), _pages(lens[b] + n, page)):
            count -= 1
            table[b][j] = free[count]
        for p in range(lens[b], lens[b] + n):
            pos.append(p)
            slots.append(table[b][p // page] * page + p % page)
        lens[b] += n
        cu.append(cu[-1] + n)
    behind = s["tokens"] - len(pos)
    return [_ints(x) for x in (lens, table, free, [count], cu, pos + [0] * behind, slots + [-1] * behind, [0])]


def _exact_store(s):
    case = s["case"]
    h, g, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    x = s["qkv"].double().view(-1, h + 2 * g, d)
    half = torch.arange(d // 2, device=x.device)
    first, second = (2 * half, 2 * half + 1) if case["paired"] else (half, half + d // 2)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]

    def turned(part, weight):
        part = part / ((part.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt()) * weight.double()
        z = torch.complex(part[..., first], part[..., second]) * turn
        y = torch.empty_like(part)
        y[..., first], y[..., second] = z.real, z.imag
        return y

    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    k = turned(x[:, h : h + g], s["norm_k"])
    at = s["slots"].long()
    real = at >= 0
    flat = lambda c: c.transpose(1, 2).reshape(-1, g, d)  # noqa: E731
    back = lambda c: c.view(-1, page, g, d).transpose(1, 2).contiguous()  # noqa: E731
    fk, fv = flat(k_pages), flat(v_pages)
    fk[at[real]], fv[at[real]] = k[real], x[:, h + g :][real]
    return [turned(x[:, :h], s["norm_q"]).reshape(-1, h * d), back(fk), back(fv)]


def _exact_attend(s):
    """Head by head: weights from the logarithm of the sum of exponentials."""
    case = s["case"]
    h, g, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    cu, totals = s["cu_tokens"].tolist(), s["key_lens"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, keys in enumerate(totals):
        n = cu[b + 1] - cu[b]
        at = torch.arange(keys, device=out.device)
        page_of, offset = s["table"][b].long()[at // page], at % page
        hidden = at[None] > (keys - n + torch.arange(n, device=out.device))[:, None]
        for c in range(g):
            k, v = s["k_pages"][page_of, c, offset].double(), s["v_pages"][page_of, c, offset].double()
            for head in range(c * (h // g), (c + 1) * (h // g)):
                logits = torch.einsum("nd,kd->nk", s["q"][cu[b] : cu[b + 1], head * d : (head + 1) * d].double(), k) / math.sqrt(d)
                if case["causal"]:
                    logits[hidden] = -math.inf
                out[cu[b] : cu[b + 1], head * d : (head + 1) * d] = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True)) @ v
    return [out]
