"""Serving and position operators next to attention, for timing and for comparing results: each call in elementary torch
operations (`own` false) and through the package's public entry points (`own` true).

  plan      block tables, slots and positions of a step, built on the GPU from request lengths: torch_mlu_amd.paged_plan
  write     new keys and values into a paged 8-bit cache with a scale per (block of tokens, head):
            torch_mlu_amd.paged_cache_write
  attend    attention over that cache: one or a few new tokens per sequence, a chunk of a long prompt, or a packed batch of
            both: torch_mlu_amd.paged_attention
  rotary    rotary positions with one or several axes, for inference and, with gradients, for training: torch_mlu_amd.rotary

A case is a dict of plain values; lengths that vary inside a batch follow from its `lens` number alone, every tensor's values
from the seed given to prepare().
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_SMALLEST = 2.0 ** -100  # of a scale


def listed():
    return [
        # a decode step of a full server: every request one token more, some need a page; pure latency
        _plan(batch=64, keys=8192, new="one", page=64, lens=1),
        # a step that mixes prompts and decodes of many requests, with more asked for than the pool has
        _plan(batch=1000, keys=4096, new="mixed", page=32, tokens=32768, short=True, lens=2),
        # the decode step's keys and values, one row into each sequence's last block
        _write(batch=64, new=1, heads=8, head_dim=128, page=64, block=64, form="e4m3", dtype="bf16", lens=3),
        # a server's prefill step: eight prompts' rows, whole blocks mostly
        _write(batch=8, new=2000, heads=8, head_dim=128, page=64, block=64, form="e4m3", dtype="bf16", lens=4),
        # the same with 8-bit integers, smaller heads and blocks, one shape a graph was captured for: padded
        _write(batch=5, new=700, heads=16, head_dim=64, page=128, block=32, form="int8", dtype="fp16", pad=200, lens=5),
        # one conversation, one token: latency
        _attend("decode", batch=1, heads=32, kv_heads=8, seq=1, keys=4097, page=64, block=64, form="e4m3", dtype="bf16", lens=6),
        # a full decode batch, every cache nearly full, bound by reading it
        _attend("decode", batch=64, heads=32, kv_heads=8, seq=1, keys=8192, page=64, block=64, form="e4m3", dtype="bf16", lens=7, full=True),
        # continuous batching with two speculative tokens, ragged fill, integers
        _attend("decode", batch=32, heads=28, kv_heads=4, seq=2, keys=5000, page=128, block=32, form="int8", dtype="fp16", lens=8),
        # chunked prefill deep in a long prompt
        _attend("chunk", batch=1, heads=32, kv_heads=8, seq=500, keys=32768, page=64, block=64, form="e4m3", dtype="bf16", lens=9),
        # prompts and decodes in one packed call
        _attend("mixed", batch=16, heads=32, kv_heads=8, seq=512, keys=4096, page=64, block=64, form="e4m3", dtype="bf16", lens=10),
        # positions of a packed serving step, one axis, far into long prompts
        _rotary("serve", batch=1, seq=2000, heads=32, kv_heads=8, head_dim=128, axes=1, dtype="bf16", far=1 << 20),
        # a training step on video tokens: time, height and width
        _rotary("train", batch=4, seq=4096, heads=16, kv_heads=16, head_dim=128, axes=3, dtype="bf16", far=4096),
    ]


def _named(case):
    c = case
    if c["kind"] == "plan":
        c["name"] = "plan_%dx%s" % (c["batch"], c["new"])
    elif c["kind"] == "write":
        c["name"] = "write_%s_%dx%d" % (c["form"], c["batch"], c["new"])
    elif c["kind"] == "attend":
        c["name"] = "%s_%s_%dx%dx%d" % (c["how"], c["form"], c["batch"], c["seq"], c["keys"])
    else:
        c["name"] = "rotary_%s_%dx%d" % (c["how"], c["batch"], c["seq"])
    return c


def _plan(*, batch, keys, new, page, lens, tokens=None, short=False):
    return _named(dict(kind="plan", batch=batch, keys=keys, new=new, page=page, lens=lens, tokens=tokens or batch, short=short))


def _write(*, batch, new, heads, head_dim, page, block, form, dtype, lens, pad=0):
    return _named(dict(kind="write", batch=batch, new=new, heads=heads, head_dim=head_dim, page=page, block=block, form=form, dtype=dtype,
                       lens=lens, pad=pad))


def _attend(how, *, batch, heads, kv_heads, seq, keys, page, block, form, dtype, lens, head_dim=128, full=False):
    return _named(dict(kind="attend", how=how, batch=batch, heads=heads, kv_heads=kv_heads, seq=seq, keys=keys, page=page, block=block,
                       form=form, dtype=dtype, lens=lens, head_dim=head_dim, full=full))


def _rotary(how, *, batch, seq, heads, kv_heads, head_dim, axes, dtype, far, interleaved=False):
    return _named(dict(kind="rotary", how=how, batch=batch, seq=seq, heads=heads, kv_heads=kv_heads, head_dim=head_dim, axes=axes,
                       dtype=dtype, far=far, interleaved=interleaved))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = ((8, 8), (16, 16), (16, 4), (32, 8), (28, 4), (16, 1))


def draw(rng):
    kind = rng.choice(("plan", "write", "write", "attend", "attend", "attend", "rotary"))
    lens = rng.randrange(1 << 20)
    page = rng.choice((32, 64, 128, 256))
    block = rng.choice([n for n in (32, 64, 128, 256) if n <= page])
    form = rng.choice(("e4m3", "int8"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if kind == "plan":
        new = rng.choice(("one", "mixed"))
        batch = _log(rng, 1, 4000)
        c = _plan(batch=batch, keys=_log(rng, 64, 16384), new=new, page=page, lens=lens, short=rng.random() < 0.25,
                  tokens=batch if new == "one" else batch + _log(rng, 64, 65536))
    elif kind == "write":
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 8000)
        c = _write(batch=_log(rng, 1, max(1, min(256, 16384 // new))), new=new, heads=rng.choice((1, 4, 8, 16)), page=page, block=block,
                   head_dim=rng.choice((64, 96, 128, 128, 256)), form=form, dtype=dtype, lens=lens, pad=rng.choice((0, 0, 17, 300)))
    elif kind == "attend":
        how = rng.choice(("decode", "decode", "chunk", "mixed"))
        heads, kv_heads = rng.choice(_HEADS)
        head_dim = rng.choice((64, 128, 128, 128, 96, 256))
        if how == "decode":
            keys = _log(rng, 40, 65536)
            seq, batch = rng.choice((1, 1, 1, 2, 3, 4, 8)), _log(rng, 1, max(1, min(128, (1 << 18) // keys)))
        elif how == "chunk":
            seq = _log(rng, 20, 1024)
            batch, keys = rng.choice((1, 1, 2)), _log(rng, max(1024, seq), 32768 if seq <= 500 else 8192)
        else:
            keys = _log(rng, 512, 4096)
            batch, seq = _log(rng, 2, 16), _log(rng, 16, 512)
        seq = min(seq, keys)
        c = _attend(how, batch=batch, heads=heads, kv_heads=kv_heads, seq=seq, keys=keys, page=page, block=block, form=form, dtype=dtype,
                    lens=lens, head_dim=head_dim)
    else:
        how = rng.choice(("serve", "train"))
        heads, kv_heads = rng.choice(_HEADS)
        seq = _log(rng, 1, 8192)
        c = _rotary(how, batch=_log(rng, 1, max(1, 8192 // seq)), seq=seq, heads=heads, kv_heads=kv_heads,
                    head_dim=rng.choice((64, 80, 128, 128, 256)), axes=rng.choice((1, 2, 3)), dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")),
                    far=rng.choice((4096, 1 << 20)), interleaved=rng.random() < 0.3)
    del c["name"]
    return c


def _requests(case):
    """(cached, new) tokens of every request."""
    r, kind = random.Random(case["lens"]), case["kind"]
    if kind == "plan":
        cached = [r.randint(1, case["keys"] - 1) for _ in range(case["batch"])]
        new = [1] * case["batch"]
        if case["new"] == "mixed":
            # every eighth request brings a prompt: together they fill the step; some are idle
            rest = case["tokens"] - case["batch"]
            for i in range(0, case["batch"], 8):
                n = min(rest, r.randint(0, 16 * case["tokens"] // case["batch"] + 16))
                cached[i], new[i], rest = r.choice((0, cached[i])), 1 + n, rest - n
            for i in range(3, case["batch"], 16):
                new[i] = 0
        return cached, new
    if kind == "write":
        cached = [r.choice((0, r.randint(0, 4 * case["page"]))) if case["new"] > 1 else r.randint(0, 4 * case["page"]) for _ in range(case["batch"])]
        return cached, [r.randint(case["new"] // 2, case["new"]) if case["new"] > 1 else 1 for _ in range(case["batch"])]
    keys, seq = case["keys"], case["seq"]
    if case["how"] == "mixed":  # a prompt's chunk in every fourth, the others decode
        new = [r.randint(seq // 2, seq) if i % 4 == 0 else 1 for i in range(case["batch"])]
        new[0] = seq
    else:
        new = [seq] * case["batch"]
    low = keys - keys // 16 if case["full"] else keys if case["how"] == "chunk" else keys // 4
    total = [max(n, r.randint(low, keys)) for n in new]
    total[0] = keys
    return [t - n for t, n in zip(total, new)], new


def _sections(case):
    n = case["head_dim"] // 2
    return {1: (n,), 2: (n // 2, n - n // 2), 3: (n - 2 * (3 * n // 8), 3 * n // 8, 3 * n // 8)}[case["axes"]]


def _prefix(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return cu


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    kind = case["kind"]
    s = {"case": case}

    def normal(*shape, dtype=_DTYPES.get(case.get("dtype"))):
        return torch.randn(shape, generator=g, device=dev, dtype=dtype)

    def ints(values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device=dev)

    if kind == "plan":
        page = case["page"]
        cached, new = _requests(case)
        width = -(-(case["keys"] + case["tokens"]) // page)
        held = [-(-c // page) for c in cached]
        need = sum(-(-(c + n) // page) - h for c, n, h in zip(cached, new, held))
        free = need // 2 if case["short"] else need + 10
        pool = torch.randperm(sum(held) + free, generator=g, device=dev).to(torch.int32)
        table = torch.full((case["batch"], width), -1, dtype=torch.int32, device=dev)
        kept = torch.arange(width, device=dev)[None, :] < ints(held)[:, None]
        table[kept] = pool[: sum(held)]
        s.update(cached=ints(cached), new=ints(new), table=table, free_pages=pool[sum(held):].clone(), free_count=ints([free]))
    elif kind == "write":
        page, block, H, D = case["page"], case["block"], case["heads"], case["head_dim"]
        cached, new = _requests(case)
        first = [c // page for c in cached]  # the pages that this call reaches
        pages = [-(-(c + n) // page) - f for c, n, f in zip(cached, new, first)]
        P, T = sum(pages) + 4, sum(new)
        order = torch.randperm(P, generator=g, device=dev)
        pos = torch.arange(T, device=dev) - torch.repeat_interleave(ints(_prefix(new)[:-1], torch.int64), ints(new, torch.int64), output_size=T)
        pos += torch.repeat_interleave(ints([c - f * page for c, f in zip(cached, first)], torch.int64), ints(new, torch.int64), output_size=T)
        base = torch.repeat_interleave(ints(_prefix(pages)[:-1], torch.int64), ints(new, torch.int64), output_size=T)
        slots = order[base + pos // page] * page + pos % page
        s["slots"] = torch.cat([slots, ints([-1] * case["pad"], torch.int64)])
        # rows of tokens and heads of different size, so that some blocks' scales grow
        size = torch.exp2(torch.randint(-2, 3, (T + case["pad"], 1, 1), generator=g, device=dev).to(_DTYPES[case["dtype"]]) / 2)
        for n in ("key", "value"):
            s[n] = normal(T + case["pad"], H, D) * size
            s[n + "_pages"], s[n + "_scales"] = _cache(case, P, H, normal)
    elif kind == "attend":
        page, Hk, D = case["page"], case["kv_heads"], case["head_dim"]
        cached, new = _requests(case)
        used = [c + n for c, n in zip(cached, new)]
        width, B, Hq = -(-max(used) // page), case["batch"], case["heads"]
        P = B * width
        s["table"] = torch.randperm(P, generator=g, device=dev).to(torch.int32).reshape(B, width)
        s["used"] = ints(used)
        for n in ("key", "value"):
            s[n + "_pages"], s[n + "_scales"] = _cache(case, P, Hk, normal)
        if case["how"] == "mixed":
            s["query"], s["cu"] = normal(sum(new), Hq, D), ints(_prefix(new))
        else:
            s["query"] = normal(B, case["seq"], Hq, D).transpose(1, 2)
    else:
        B, S, D, A = case["batch"], case["seq"], case["head_dim"], case["axes"]
        sec = _sections(case)
        s["axes"] = ints([a for a, n in enumerate(sec) for _ in range(n)])
        s["freq"] = torch.tensor([10000.0 ** (-i / (D // 2)) for i in range(D // 2)], dtype=torch.float64, device=dev)
        for n, H in (("query", case["heads"]), ("key", case["kv_heads"])):
            if case["how"] == "serve":  # packed tokens of a serving step
                s[n] = normal(B * S, H, D)
            else:
                s[n] = normal(B, S, H, D).transpose(1, 2).requires_grad_()
                s["d" + n] = normal(B, S, H, D).transpose(1, 2)
        shape = (A, B * S) if case["how"] == "serve" else (A, B, S)
        s["positions"] = torch.randint(0, case["far"], shape, generator=g, device=dev, dtype=torch.int32)
    return s


def _cache(case, pages, heads, normal):
    """Pages of a cache in use, and their scales."""
    page, block, D = case["page"], case["block"], case["head_dim"]
    out = torch.empty(pages, page, heads, D, dtype=_FORMATS[case["form"]], device="cuda")
    for i in range(0, pages, 1024):
        n = min(1024, pages - i)
        x = normal(n, page, heads, D, dtype=torch.float16)
        out[i:i + n] = (x * 100).clamp_(-448, 448).to(out.dtype) if case["form"] == "e4m3" else (x * 30).round_().clamp_(-127, 127).to(out.dtype)
    step = torch.exp2(normal(pages, page // block, heads, dtype=torch.float32).mul_(0.7).round_())  # powers of two, as paged_cache_write leaves them
    return out, step * 2.0 ** -7 if case["form"] == "e4m3" else step * (1.1 / 30)


# ---- the operators --------------------------------------------------------------------------------------------------
def run(s):
    kind = s["case"]["kind"]
    return {"plan": _run_plan, "write": _run_write, "attend": _run_attend, "rotary": _run_rotary}[kind](s)


def _run_plan(s):
    case = s["case"]
    if own:
        import torch_mlu_amd

        p = torch_mlu_amd.paged_plan(s["cached"], s["new"], s["table"], s["free_pages"], s["free_count"], page_size=case["page"],
                                     max_tokens=case["tokens"])
        return {"table": s["table"], "cu": p.cu_seqlens, "used": p.seqused_k, "positions": p.positions, "slots": p.slots,
                "admitted": p.admitted, "free": p.free_count}
    page, T, table = case["page"], case["tokens"], s["table"]
    width = table.shape[1]
    cached, new = s["cached"].long().clamp(min=0), s["new"].long().clamp(min=0)
    end = new.cumsum(0)
    held, total = (cached + page - 1) // page, (cached + new + page - 1) // page
    fits = (end <= T) & (cached + new <= width * page)
    need = torch.where(fits, total - held, 0)
    taken = need.cumsum(0)
    admitted = fits & ((need == 0) | (taken <= s["free_count"]))
    j = torch.arange(width, device=table.device)[None, :]
    fill = admitted[:, None] & (j >= held[:, None]) & (j < total[:, None])
    source = s["free_count"] - 1 - ((taken - need)[:, None] + j - held[:, None])
    table.copy_(torch.where(fill, s["free_pages"][source.clamp(0, s["free_pages"].numel() - 1)] if s["free_pages"].numel() else table, table))
    t = torch.arange(T, device=table.device)
    b = torch.searchsorted(end, t, right=True)
    real = b < new.numel()
    b = b.clamp(max=new.numel() - 1)
    pos = torch.where(real, cached[b] + t - (end - new)[b], 0)
    entry = table[b, (pos // page).clamp(max=width - 1)].long()
    slots = torch.where(real & admitted[b] & (entry >= 0), entry * page + pos % page, -1)
    free = s["free_count"] - torch.where(admitted & (need > 0), taken, 0).max()
    cu = torch.cat([end.new_zeros(1), end.clamp(max=T)])
    return {"table": table, "cu": cu.int(), "used": torch.where(admitted, cached + new, cached).int(), "positions": pos.int(), "slots": slots,
            "admitted": admitted, "free": free.int()}


def _run_write(s):
    if own:
        import torch_mlu_amd

        torch_mlu_amd.paged_cache_write(s["key"], s["value"], s["key_pages"], s["value_pages"], s["key_scales"], s["value_scales"], s["slots"])
    else:
        _plain_write(s["key"], s["key_pages"], s["key_scales"], s["slots"])
        _plain_write(s["value"], s["value_pages"], s["value_scales"], s["slots"])
    return {n: _held(s, n) if n.endswith("pages") else s[n] for n in ("key_pages", "value_pages", "key_scales", "value_scales")}


def _held(s, name):
    pages = s[name]
    if pages.dtype != torch.int8:
        return pages  # floating values already
    P, page, H, D = pages.shape
    scales = s[name.replace("pages", "scales")]
    return pages.view(P, scales.shape[1], -1, H, D) * scales[:, :, None, :, None]


def _plain_write(x, pages, scales, slots):
    P, page, H, D = pages.shape
    block = page // scales.shape[1]
    kept = slots >= 0
    at, x = slots[kept], x[kept].float()
    unit = at // block
    size = torch.where(x.isfinite(), x.abs(), 0).amax(-1)
    top = torch.zeros(P * page // block, H, device=x.device).index_reduce_(0, unit, size, "amax")
    ones = torch.ones_like(at, dtype=torch.float32)
    zero = torch.zeros(P * page // block, device=x.device)
    touched = zero.index_add(0, unit, ones) > 0
    fresh = zero.index_add(0, unit, (at % block == 0).float()) > 0
    old = scales.view(-1, H)
    if pages.dtype == torch.int8:
        needed = (top * (1.0 / 127)).clamp(min=_SMALLEST)
    else:
        part, power = torch.frexp(top)  # top = part 2^power with part in [1/2, 1): 448 = 7/8 2^9
        power = (power - 9 + (part > 0.875)).clamp(min=-100)
        needed = torch.where(top > 0, torch.ldexp(torch.ones_like(top), power), _SMALLEST)
    scale = torch.maximum(torch.where(fresh[:, None], 0.0, old), needed)
    again = (touched & ~fresh)[:, None] & (scale > old)

    def stored(values):
        if pages.dtype == torch.int8:
            return values.nan_to_num(nan=0.0).round().clamp(-127, 127).to(pages.dtype)
        return values.clamp(-448, 448).to(pages.dtype)

    rows = pages.view(-1, block, H, D)
    rows.copy_(torch.where(again[:, None, :, None], stored(rows.float() * (old / scale)[:, None, :, None]).float(), rows.float()).to(pages.dtype))
    old.copy_(torch.where(touched[:, None], scale, old))
    flat = pages.view(-1, H, D)
    flat.view(torch.uint8)[at] = stored(x * torch.reciprocal(scale)[unit][:, :, None]).view(torch.uint8)


def _run_attend(s):
    case = s["case"]
    mixed = case["how"] == "mixed"
    if own:
        import torch_mlu_amd

        more = dict(cu_seqlens_q=s["cu"], max_seqlen_q=case["seq"]) if mixed else {}
        return torch_mlu_amd.paged_attention(s["query"], s["key_pages"], s["value_pages"], s["table"], s["used"], is_causal=True,
                                             key_scales=s["key_scales"], value_scales=s["value_scales"], **more)
    q = s["query"]
    B, S, Hq, Hk, D = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"]
    dev = q.device
    if mixed:
        cu = s["cu"].long()
        rows = cu[1:] - cu[:-1]
        at = cu[:-1, None] + torch.arange(S, device=dev)[None, :]
        real = torch.arange(S, device=dev)[None, :] < rows[:, None]
        qp = q[at.clamp(max=q.shape[0] - 1)].transpose(1, 2)
    else:
        rows, qp = torch.full((B,), S, device=dev), q

    def gathered(pages, scales):
        index = s["table"].long()
        x = pages.view(torch.uint8)[index].view(pages.dtype).float()  # [B, pages, page, Hk, D]
        sc = scales[index]
        x = x.view(*sc.shape[:3], -1, Hk, D).mul_(sc[:, :, :, None, :, None])
        return x.view(B, -1, Hk, D)

    k = gathered(s["key_pages"], s["key_scales"]).permute(0, 2, 3, 1).contiguous()
    score = torch.matmul(qp.float().reshape(B, Hk, Hq // Hk * S, D), k).view(B, Hq, S, -1).mul_(1.0 / math.sqrt(D))
    del k
    used = s["used"].long()
    last = (used - rows)[:, None] + torch.arange(S, device=dev)[None, :]  # [B, S]: the last key that a row sees
    hidden = torch.arange(score.shape[-1], device=dev)[None, None, :] > torch.minimum(last, used[:, None] - 1)[:, :, None]
    score.masked_fill_(hidden[:, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp_(min=torch.finfo(torch.float32).min)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = gathered(s["value_pages"], s["value_scales"]).permute(0, 2, 1, 3).contiguous()
    out = torch.matmul(p.view(B, Hk, Hq // Hk * S, -1), v).view(B, Hq, S, D)
    out = torch.where(total > 0, out / total, 0).to(q.dtype)
    lse = torch.where(total > 0, top + total.log(), float("inf"))[..., 0]
    if mixed:
        return out.transpose(1, 2)[real], lse.transpose(1, 2)[real].t().contiguous()
    return out, lse


def _run_rotary(s):
    case = s["case"]
    train = case["how"] == "train"
    if own:
        import torch_mlu_amd

        q, k = torch_mlu_amd.rotary(s["query"], s["key"], s["positions"], s["freq"], s["axes"], interleaved=case["interleaved"])
        if not train:
            return q, k
        return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (s["query"], s["key"]), (s["dquery"], s["dkey"]))
    # angles of far positions in 64 bits
    pos = s["positions"][s["axes"].long()].movedim(0, -1).unsqueeze(-3 if not train else -2)
    angle = pos.double() * s["freq"]  # [B, S, 1, n] or [1, T, n]
    angle = angle.transpose(1, 2) if train else angle.transpose(0, 1)
    cos, sin = angle.cos().float(), angle.sin().float()

    def turned(x, sin):
        y = x.detach().float()
        if case["interleaved"]:
            a, b = y[..., 0::2], y[..., 1::2]
            return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2).to(x.dtype)
        a, b = y.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(x.dtype)

    out = (turned(s["query"], sin), turned(s["key"], sin))
    return out + (turned(s["dquery"], -sin), turned(s["dkey"], -sin)) if train else out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "plan":
        cached, new = _requests(case)
        page = case["page"]
        pages = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, new))
        # lengths in, prefix sums, fill and admission out, new pages from the list into the table, positions and slots out
        return {"bytes": 17.0 * case["batch"] + 8.0 * pages + 12.0 * case["tokens"], "flops": 0.0}
    if kind == "write":
        _, new = _requests(case)
        values = 2.0 * sum(new) * case["heads"] * case["head_dim"]
        return {"bytes": 3.0 * values + 8.0 * (sum(new) + case["pad"]) + 8.0 * values / case["head_dim"] / case["block"], "flops": 0.0}
    if kind == "attend":
        cached, new = _requests(case)
        Hq, Hk, D = case["heads"], case["kv_heads"], case["head_dim"]
        keys, rows = sum(cached) + sum(new), sum(new)
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, new))
        size = 2.0 * keys * Hk * D + 8.0 * keys * Hk / case["block"] + 4.0 * rows * Hq * D + 4.0 * rows * Hq + 4.0 * keys / case["page"]
        return {"bytes": size, "flops": 4.0 * Hq * D * pairs}
    rows = case["batch"] * case["seq"]
    values = rows * (case["heads"] + case["kv_heads"]) * case["head_dim"]
    passes = 2 if case["how"] == "train" else 1
    size = 4.0 if case["dtype"] == "fp32" else 2.0
    return {"bytes": passes * (2.0 * size * values + 4.0 * rows * case["axes"]), "flops": passes * 3.0 * values}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "write": _exact_write, "attend": _exact_attend, "rotary": _exact_rotary}[case["kind"]](s)


def _exact_plan(s):
    case = s["case"]
    page, T = case["page"], case["tokens"]
    cached, new, table, pool = (s[n].cpu().numpy().astype(np.int64) for n in ("cached", "new", "table", "free_pages"))
    free, cu = int(s["free_count"]), [0]
    wanted, left = 0, free
    pos, slots, used, admitted = np.zeros(T, np.int64), np.full(T, -1, np.int64), cached.copy(), np.zeros(len(new), bool)
    for b in range(len(new)):
        cu.append(cu[-1] + int(new[b]))
        have, want = -(-int(cached[b]) // page), -(-int(cached[b] + new[b]) // page)
        fits = cu[-1] <= T and want <= table.shape[1] and cached[b] + new[b] <= table.shape[1] * page
        first = wanted
        wanted += want - have if fits else 0
        admitted[b] = fits and (want == have or wanted <= free)
        at = np.arange(cu[b], min(cu[b + 1], T))
        pos[at] = cached[b] + at - cu[b]
        if admitted[b]:
            table[b, have:want] = pool[free - 1 - first - np.arange(want - have)]
            left = free - wanted if want > have else left
            used[b] += new[b]
            slots[at] = table[b, pos[at] // page] * page + pos[at] % page
    return {"table": table, "cu": np.minimum(np.array(cu), T), "used": used, "positions": pos, "slots": slots, "admitted": admitted,
            "free": np.array([left])}


def _exact_write(s):
    """Eight-bit integers have no value here: which whole step a quotient next to a half goes to is the rounding's choice."""
    whole = s["case"]["form"] == "int8"
    out = {}
    slots = s["slots"].cpu().numpy()
    for n in ("key", "value"):
        pages, scales, x = s[n + "_pages"].double(), s[n + "_scales"].double(), s[n].double()
        P, page, H, D = pages.shape
        block = page // scales.shape[1]
        rows, old = pages.view(-1, block, H, D), scales.view(-1, H)
        begin = 0
        while begin < len(slots):
            unit, end = slots[begin] // block, begin + 1
            while end < len(slots) and slots[end] // block == unit:
                end += 1
            if slots[begin] >= 0:
                y = x[begin:end]
                top = y.abs().amax((0, 2))
                need = (top / 127).clamp(min=_SMALLEST) if whole else torch.exp2(torch.log2(top / 448).ceil().clamp(min=-100))
                before = torch.zeros_like(need) if slots[begin] % block == 0 else old[unit].clone()
                now = torch.maximum(before, need)
                if slots[begin] % block and not whole:
                    rows[unit] = _to_e4m3(rows[unit] * (before / now)[:, None])
                old[unit] = now
                if not whole:
                    first = int(slots[begin] % block)
                    rows[unit, first:first + end - begin] = _to_e4m3(y / now[:, None])
            begin = end
        out[n + "_pages"], out[n + "_scales"] = None if whole else pages, scales
    return out


def _to_e4m3(x):
    step = torch.exp2(torch.log2(x.abs().clamp(min=2.0 ** -6)).floor() - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_attend(s):
    case = s["case"]
    B, S, Hq, Hk, D, page = case["batch"], case["seq"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    mixed = case["how"] == "mixed"
    cu = s["cu"].tolist() if mixed else None
    used, q = s["used"].tolist(), s["query"].double()
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.zeros((Hq, q.shape[0]) if mixed else (B, Hq, S), dtype=torch.float64, device=q.device)
    for b in range(B):
        n = used[b]
        kv = []
        for name in ("key", "value"):
            index = s["table"][b, : -(-n // page)].long()
            x = s[name + "_pages"].view(torch.uint8)[index].view(s[name + "_pages"].dtype).double().flatten(0, 1)[:n]
            kv.append(x * s[name + "_scales"].double()[index].flatten(0, 1).repeat_interleave(case["block"], 0)[:n, :, None])
        rows = q[cu[b]:cu[b + 1]] if mixed else q[b].transpose(0, 1)
        L = rows.shape[0]
        seen = torch.ones(L, n, dtype=torch.bool, device=q.device).tril(n - L)
        for h in range(Hq):
            x = (rows[:, h] @ kv[0][:, h * Hk // Hq].t().contiguous()) / math.sqrt(D)
            x = torch.where(seen, x, -torch.inf)
            z = torch.logsumexp(x, -1)
            o = torch.exp(x - z[:, None]) @ kv[1][:, h * Hk // Hq].contiguous()
            if mixed:
                out[cu[b]:cu[b + 1], h], lse[h, cu[b]:cu[b + 1]] = o, z
            else:
                out[b, h], lse[b, h] = o, z
    return out, lse


def _exact_rotary(s):
    case = s["case"]
    n, train = case["head_dim"] // 2, case["how"] == "train"
    axes, freq = s["axes"].tolist(), s["freq"].tolist()
    out = []
    for name in ("query", "key") + (("dquery", "dkey") if train else ()):
        x = s[name].detach().double()
        y = torch.empty_like(x)
        for i in range(n):
            t = s["positions"][axes[i]].double() * freq[i] * (-1.0 if name[0] == "d" else 1.0)
            t = t[:, None, :] if train else t[:, None]
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + n)
            z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.ones_like(t), t)
            y[..., a], y[..., b] = z.real, z.imag
        out.append(y)
    return tuple(out)
