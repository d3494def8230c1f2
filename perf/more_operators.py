"""Attention over whole prompts and the 4-bit KV cache as cases that can be timed and
compared: a packed batch of prompts attended, new tokens written to the cache (with the
norms of queries and keys and the position rotation in the same pass), the cache read
back, and attention of new tokens over it.

  own         False: `run` computes the plain form; True: it calls the package
  listed()    the cases that stand for the range
  draw(rng)   one more case of the same range
  prepare     the activations, the page pool and the page table a serving loop holds
  run         one call, and what it gives
  work        bytes and flops one call cannot do without
  exact       what `run` gives, from the definition in 64 bits

Definitions.  Prompts: row i of a sequence of n new tokens and m keys attends keys
0 .. m - n + i; with none of them its output is zero, as are rows of no sequence.  Cache:
every 32 consecutive values of a row of K or V have an fp16 scale s and offset m, and a
code c, 0 .. 15, stands for c * s + m; s = (max - min) / 15 and m = min of the 32 values,
rounded to fp16, and c the integer nearest to (x - m) / s (zero where s is).
"""
from __future__ import annotations

import math

import torch

own = False

_BLOCKS, _BLOCK_INDEX = 2, 1  # transformer blocks in a page, the block called
_GROUP = 32                   # values of a scale
_EPS = 1e-5
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _case(name, op, bs, positions, new=1, dtype="bf16", heads=32, kv_heads=8, head_dim=128, stride=32, norm=False,
          order="pairs", softcap=0.0, behind=0):
    """positions: cached positions of the longest sequence before the call (prompt, write) or in
    all (read, attend); new: new tokens of the longest sequence; behind: rows of no sequence."""
    return {"name": name, "op": op, "bs": bs, "positions": positions, "new": new, "dtype": dtype, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "stride": stride, "norm": norm, "order": order, "softcap": softcap,
            "behind": behind}


def listed():
    return [
        # one short chat turn: launch latency
        _case("prompt_1x17", "prompt", 1, 0, new=17),
        # a prefill batch of ragged prompts, the widest configuration with its softcap, a padded buffer
        _case("prompt_16x1500_f16_cap", "prompt", 16, 0, new=1500, dtype="f16", heads=48, softcap=30.0, behind=37),
        # one long document
        _case("prompt_1x8192", "prompt", 1, 0, new=8192),
        # short follow-ups to long cached prompts: few rows, long keys
        _case("prompt_4x60_after_16000", "prompt", 4, 16000, new=60),
        # 32-bit activations, small heads
        _case("prompt_6x777_f32", "prompt", 6, 0, new=777, dtype="f32", heads=16, kv_heads=4, head_dim=64),
        # a decode step of the largest batch
        _case("write_64x1_norm", "write", 64, 4000, norm=True),
        # a batch of ragged prompts, half-split rotation, queries and keys normed
        _case("write_3x777_norm_halves", "write", 3, 0, new=777, norm=True, order="halves"),
        # the cached prefix of one short prompt, small heads
        _case("read_1x333_f16", "read", 1, 333, dtype="f16", heads=16, kv_heads=4, head_dim=64, stride=16),
        # the cached prefixes of a full batch
        _case("read_32x4000", "read", 32, 4000),
        # one decode step of one short sequence: launch latency
        _case("attend_1x100", "attend", 1, 100),
        # the ordinary decode batch
        _case("attend_32x4000", "attend", 32, 4000),
        # five drafted tokens of each sequence checked at once, the widest configuration with its softcap
        _case("attend_8x8190_new5_f16_cap", "attend", 8, 8190, new=5, dtype="f16", heads=48, softcap=30.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "prompt", "write", "read", "attend", "attend"])
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (48, 8, 128), (16, 4, 64), (8, 1, 128), (8, 8, 64)])
    c = dict(dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
             stride=rng.choice([16, 32, 32, 64]))
    bs, new, positions = _log_int(rng, 1, 64), 1, _log_int(rng, 16, 8192)
    if op == "prompt":
        c.update(softcap=rng.choice([0.0, 0.0, 30.0]), behind=rng.choice([0, 0, rng.randint(1, 100)]))
        new, positions = _log_int(rng, 1, 8192), rng.choice([0, 0, _log_int(rng, 1, 16000)])
        rows, pairs = 16384, 8192 * 8192 // 2 * 32 * 128 // (heads * head_dim)
        if c["dtype"] == "f32":
            rows, new, positions = 8192, min(new, 2048), min(positions, 4096)
        new = min(new, int((2 * pairs) ** 0.5))
        positions = min(positions, max(0, pairs // new - new // 2 - 1))
        bs = max(1, min(bs, rows // new, pairs // (new * (new // 2 + positions) + 1), 4 * rows // (new + positions)))
    elif op == "write":
        c.update(norm=rng.random() < 0.5, order=rng.choice(["pairs", "halves"]))
        if rng.random() < 0.5:  # a prompt batch
            new, positions = _log_int(rng, 2, 2048), rng.choice([0, 0, rng.randint(1, 2000)])
            bs = max(1, min(bs, 2400 // new))
    elif op == "read":
        bs = max(1, min(bs, 32 * 4000 // positions))
    else:
        new, positions = rng.choice([1, 1, 1, rng.randint(2, 8)]), _log_int(rng, 16, 32768)
        bs = max(1, min(bs, 32 * 4000 // positions // (1 if new == 1 else 2)))
        c.update(softcap=rng.choice([0.0, 0.0, 30.0]))
        positions = max(positions, 2 * new)
    got = _case("", op, bs, positions, new, **c)
    del got["name"]
    return got


def _lengths(case):
    """Ragged over the batch, between half of `positions` and all of it."""
    bs, n = case["bs"], case["positions"]
    return [n - (i * (n // 2)) // bs for i in range(bs)]


def _new_lengths(case):
    """New tokens of each sequence: prompts are ragged, decode steps are not."""
    bs, n = case["bs"], case["new"]
    return [n - (i * (n // 2)) // bs for i in range(bs)] if n > 16 else [n] * bs


def _starts(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------ inputs
def _quantise(x):
    """x [..., hd] fp32 -> codes [..., hd] as numbers and (scale, offset) [..., hd / 32, 2] fp16, quotients in 64 bits."""
    y = x.unflatten(-1, (-1, _GROUP))
    lo, hi = y.amin(-1), y.amax(-1)
    s, m = ((hi - lo) / 15.0).half(), lo.half()
    q = (y.double() - m.double()[..., None]) / s.double()[..., None]
    c = torch.where(s[..., None] > 0, q, 0.0).round().clamp(0, 15)
    return c.flatten(-2).to(torch.uint8), torch.stack([s, m], dim=-1)


def _pack(c):
    """Two codes a byte, the even element in the low half."""
    return c[..., 0::2] | c[..., 1::2] << 4


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    bs, new, heads, kvh, hd, stride = (case[k] for k in ("bs", "new", "heads", "kv_heads", "head_dim", "stride"))
    dtype = _DT[case["dtype"]]
    lens, news = _lengths(case), _new_lengths(case)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    s = {"case": case}
    if case["op"] == "prompt":
        # queries of a standard deviation that gives scores one of 1.5
        rows = sum(news) + case["behind"]
        if case["positions"]:  # a continued prompt: keys and values gathered from the cache and the new tokens
            s["q"] = (rn(rows, heads, hd) * 1.5).to(dtype)
            keys = sum(lens) + sum(news) + case["behind"]
            s["k"], s["v"] = rn(keys, kvh, hd).to(dtype), rn(keys, kvh, hd).to(dtype)
        else:  # views of one fused projection's output
            qkv = rn(rows, (heads + 2 * kvh) * hd)
            qkv[:, : heads * hd] *= 1.5
            q, k, v = qkv.to(dtype).split([heads * hd, kvh * hd, kvh * hd], dim=-1)
            s["q"], s["k"], s["v"] = q.unflatten(-1, (heads, hd)), k.unflatten(-1, (kvh, hd)), v.unflatten(-1, (kvh, hd))
        s["cu_q"] = _starts(news)
        s["cu_k"] = _starts([n + m for n, m in zip(lens, news)])
        return s
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    # the page pool, with quantised values everywhere; scores of standard deviation about 1.5
    per_seq = -(-(case["positions"] + (new if case["op"] == "write" else 0)) // stride)
    pages = bs * per_seq + 1
    s["ids"] = (1 + torch.randperm(pages - 1, generator=gen, device="cuda")).view(bs, per_seq).to(torch.int32)
    slab = torch.zeros(pages, _BLOCKS, kvh, 2, stride, hd // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(pages, _BLOCKS, kvh, 2, stride, hd // _GROUP, 2, dtype=torch.float16, device="cuda")
    codes, scales[:, _BLOCK_INDEX] = _quantise(rn(pages, kvh, 2, stride, hd) * 1.5)
    slab[:, _BLOCK_INDEX] = _pack(codes)
    s["state"] = [slab.flatten(1), scales.flatten(1)]
    del codes
    if case["op"] == "write":
        # one fused projection's output: q, k and v are views of it; without rare large values
        qkv = rn(bs, new, (heads + 2 * kvh) * hd).clamp_(-2.5, 2.5).to(dtype)
        q, k, v = qkv.split([heads * hd, kvh * hd, kvh * hd], dim=-1)
        s["q"], s["k"], s["v"] = q.unflatten(-1, (heads, hd)), k.unflatten(-1, (kvh, hd)), v.unflatten(-1, (kvh, hd))
        s["freqs"] = (1.0 / (10000.0 ** (torch.arange(0, hd, 2).float() / hd))).cuda()
        s["q_norm"] = 1.0 + 0.1 * rn(hd) if case["norm"] else None
        s["k_norm"] = 1.0 + 0.1 * rn(hd) if case["norm"] else None
        s["new_lens"] = torch.tensor(news, dtype=torch.int32, device="cuda") if new > 16 else None
        # the pages this call writes to, and how far they are filled after it
        first = [n // stride for n in lens]
        most = max((n + m - 1) // stride - f + 1 for n, m, f in zip(lens, news, first))
        at = torch.tensor(first, device="cuda")[:, None] + torch.arange(most, device="cuda")
        s["tail_ids"] = s["ids"].gather(1, at.clamp(max=per_seq - 1))
        s["tail_lens"] = torch.tensor([n + m - f * stride for n, m, f in zip(lens, news, first)], dtype=torch.int32,
                                      device="cuda")
    elif case["op"] == "attend":
        s["q"] = rn(bs, new, heads, hd).to(dtype)
    if own:  # the handle of the package's cache, kept for the model's life
        from shark_platform_b200 import attention as A

        s["cache"] = A.PagedKVCache(transformer_block_count=_BLOCKS, attn_head_count=kvh, attn_head_dim=hd,
                                    block_seq_stride=stride, dtype=torch.uint8, device="cuda")
    return s


# ------------------------------------------------------------------------ plain form
def _softmax_values(w, dead, v):
    """w [bs, kv_heads, group, rows, keys] scores, dead [bs, rows, keys]; v [bs, kv_heads, keys, hd]."""
    w = w.masked_fill_(dead[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    p = w.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, w.shape[2:4])
    return torch.where(total > 0, o / total, 0.0)


def _scores(q, k, case):
    """q [bs, kv_heads, rows, hd], k [bs, kv_heads, keys, hd], fp32."""
    w = torch.matmul(q, k.transpose(-1, -2)).mul_(case["head_dim"] ** -0.5)
    return w.div_(case["softcap"]).tanh_().mul_(case["softcap"]) if case["softcap"] else w


def _plain_prompt(s):
    case = s["case"]
    heads, kvh, hd = case["heads"], case["kv_heads"], case["head_dim"]
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    len_q, len_k = cu_q.diff()[:, None], cu_k.diff()[:, None]
    i = torch.arange(case["new"], device="cuda")
    j = torch.arange(case["new"] + case["positions"], device="cuda")
    live_q, live_k = i < len_q, j < len_k
    at_q, at_k = torch.where(live_q, cu_q[:-1, None] + i, 0), torch.where(live_k, cu_k[:-1, None] + j, 0)
    # the batch padded: [bs, kv_heads, group * rows, hd] and [bs, kv_heads, keys, hd]
    q = s["q"][at_q].float().unflatten(2, (kvh, heads // kvh)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = (torch.where(live_k[..., None, None], x[at_k].float(), 0.0).transpose(1, 2) for x in (s["k"], s["v"]))
    dead = j > (len_k - len_q + i)[..., None]
    o = _softmax_values(_scores(q, k, case).unflatten(2, (heads // kvh, -1)), dead, v)
    out = torch.zeros(s["q"].shape, dtype=s["q"].dtype, device="cuda")
    out[at_q[live_q]] = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[live_q].to(out.dtype)
    return out


def _rotate(x, pos, s, weight, case):
    """x [bs, new, heads, hd] fp32, pos [bs, new]: normed and rotated; angles in 64 bits."""
    if weight is not None:
        x = weight * (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS))
    a = pos[..., None].double() * s["freqs"].double()
    cos, sin = a.cos().float()[:, :, None], a.sin().float()[:, :, None]
    if case["order"] == "halves":
        re, im = x.chunk(2, dim=-1)
        return torch.cat([re * cos - im * sin, im * cos + re * sin], dim=-1)
    re, im = x[..., 0::2], x[..., 1::2]
    return torch.stack([re * cos - im * sin, im * cos + re * sin], dim=-1).flatten(-2)


def _views(s):
    case = s["case"]
    dims = (_BLOCKS, case["kv_heads"], 2, case["stride"])
    hd = case["head_dim"]
    return s["state"][0].unflatten(1, dims + (hd // 2,)), s["state"][1].unflatten(1, dims + (hd // _GROUP, 2))


def _read(s, ids, lens):
    """K and V of the listed pages, [2, bs, positions, kv_heads, hd] fp32, zero at and behind `lens`."""
    slab, scales = _views(s)
    c = slab[:, _BLOCK_INDEX][ids.long()]                       # [bs, n, heads, 2, stride, hd / 2]
    f = scales[:, _BLOCK_INDEX][ids.long()].float()[..., None]  # [bs, n, heads, 2, stride, hd / 32, 2, 1]
    c = torch.stack([c & 15, c >> 4], dim=-1).flatten(-2).float().unflatten(-1, (-1, _GROUP))
    x = (c * f[..., 0, :] + f[..., 1, :]).flatten(-2).permute(3, 0, 1, 4, 2, 5).flatten(2, 3)
    live = torch.arange(x.shape[2], device=x.device) < lens[:, None]
    return torch.where(live[None, :, :, None, None], x, 0.0)


def _plain_write(s):
    case = s["case"]
    dtype, stride = _DT[case["dtype"]], case["stride"]
    i = torch.arange(case["new"], device="cuda")
    pos = s["lens"].long()[:, None] + i
    q = _rotate(s["q"].float(), pos, s, s["q_norm"], case).to(dtype)
    k = _rotate(s["k"].float(), pos, s, s["k_norm"], case)
    codes, scales = _quantise(torch.stack([k, s["v"].float()], dim=3))  # [bs, new, heads, 2, ..]
    slab, held = _views(s)
    live = (i < (case["new"] if s["new_lens"] is None else s["new_lens"][:, None])).expand_as(pos)
    page = s["ids"].long().gather(1, pos // stride)[live]
    slab[page, _BLOCK_INDEX, :, :, pos[live] % stride] = _pack(codes)[live]
    held[page, _BLOCK_INDEX, :, :, pos[live] % stride] = scales[live]
    kc, vc = _read(s, s["tail_ids"], s["tail_lens"]).bfloat16()
    return {"q": q, "k": k.to(dtype), "k_cache": kc, "v_cache": vc}


def _plain_attend(s):
    case = s["case"]
    k, v = _read(s, s["ids"], s["lens"]).transpose(2, 3)
    bs, new, heads, hd = s["q"].shape
    kvh = case["kv_heads"]
    q = s["q"].float().view(bs, new, kvh, heads // kvh, hd).permute(0, 2, 3, 1, 4).flatten(2, 3)
    last = s["lens"][:, None] - new + torch.arange(new, device="cuda")
    dead = torch.arange(k.shape[2], device="cuda") > last[..., None]
    o = _softmax_values(_scores(q, k, case).unflatten(2, (heads // kvh, new)), dead, v)
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3).to(s["q"].dtype)


# ------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        if op == "prompt":
            return _plain_prompt(s)
        if op == "write":
            return _plain_write(s)
        if op == "read":
            k, v = _read(s, s["ids"], s["lens"]).to(_DT[case["dtype"]])
            return {"k": k, "v": v}
        return _plain_attend(s)
    from shark_platform_b200 import attention as A

    if op == "prompt":
        return A.prompt_attend(s["q"], s["k"], s["v"], cu_seqlens=s["cu_q"],
                               cu_seqlens_k=s["cu_k"] if case["positions"] else None, softcap=case["softcap"] or None)
    cache, state = s["cache"], s["state"]
    if op == "write":
        q, k = A.norm_rope_kv_write(s["q"], s["k"], s["v"], cache, state, block_index=_BLOCK_INDEX,
                                    seq_block_ids=s["ids"], start_positions=s["lens"], new_lens=s["new_lens"],
                                    freqs=s["freqs"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=_EPS,
                                    use_hf=case["order"] == "halves")
        # the values the written pages now stand for: what a continued prompt attends
        kc, vc = A.kv_read(cache, state, block_index=_BLOCK_INDEX, seq_block_ids=s["tail_ids"], seq_lens=s["tail_lens"])
        return {"q": q, "k": k, "k_cache": kc, "v_cache": vc}
    if op == "read":
        k, v = A.kv_read(cache, state, block_index=_BLOCK_INDEX, seq_block_ids=s["ids"], seq_lens=s["lens"],
                         dtype=_DT[case["dtype"]])
        return {"k": k, "v": v}
    return A.kv_attend(s["q"], cache, state, block_index=_BLOCK_INDEX, seq_block_ids=s["ids"], seq_lens=s["lens"],
                       softcap=case["softcap"] or None)


def work(case):
    bs, new, heads, kvh, hd, stride = (case[k] for k in ("bs", "new", "heads", "kv_heads", "head_dim", "stride"))
    io = 4 if case["dtype"] == "f32" else 2
    lens, news = _lengths(case), _new_lengths(case)
    held = kvh * 2 * (hd // 2 + hd // _GROUP * 4)  # codes, scales and offsets of a position
    if case["op"] == "prompt":
        pairs = sum(m * n + m * (m + 1) // 2 for n, m in zip(lens, news))
        rows = 2 * sum(news) * heads + case["behind"] * heads + 2 * (sum(lens) + sum(news)) * kvh
        return {"bytes": rows * hd * io, "flops": 4 * pairs * heads * hd}
    if case["op"] == "write":
        # q, k, v read; q and k written (padding rows too); the written pages read back as bf16 rows
        tail = [n % stride + m for n, m in zip(lens, news)]
        rows = bs * max(-(-t // stride) for t in tail) * stride
        return {"bytes": bs * new * hd * io * (2 * heads + 3 * kvh) + (sum(news) + sum(tail)) * held + rows * 4 * kvh * hd,
                "flops": bs * new * (heads + kvh) * hd * 8}
    if case["op"] == "read":
        rows = bs * -(-case["positions"] // stride) * stride
        return {"bytes": sum(lens) * held + rows * 2 * kvh * hd * io, "flops": 4 * sum(lens) * kvh * hd}
    attended = sum(n - new + 1 + i for n in lens for i in range(new))
    return {"bytes": sum(lens) * held + 2 * bs * new * heads * hd * io, "flops": 4 * attended * heads * hd}


# ------------------------------------------------------------------------ 64 bits
def _attend64(q, k, v, case):
    """One sequence in 64 bits: q [rows, heads, hd], k and v [keys, kv_heads, hd]; row i sees keys 0 .. keys - rows + i."""
    n, m = q.shape[0], k.shape[0]
    group = case["heads"] // case["kv_heads"]
    unseen = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for h in range(case["heads"]):
        w = q[:, h].double() @ k[:, h // group].double().T / math.sqrt(case["head_dim"])
        if case["softcap"]:
            w = torch.tanh(w / case["softcap"]) * case["softcap"]
        w[unseen] = -math.inf
        out[:, h] = torch.softmax(w, dim=-1) @ v[:, h // group].double()
    return out


def _cached64(s, slot, pages):
    """K (slot 0) or V (1) of a list of pages, [positions, kv_heads, hd]."""
    slab, scales = _views(s)
    b = slab[pages, _BLOCK_INDEX, :, slot].transpose(1, 2).flatten(0, 1)                # [positions, heads, hd / 2]
    f = scales[pages, _BLOCK_INDEX, :, slot].transpose(1, 2).flatten(0, 1).double()     # [positions, heads, hd / 32, 2]
    x = torch.empty(*b.shape[:2], b.shape[2] * 2, dtype=torch.float64, device=b.device)
    x[..., 0::2], x[..., 1::2] = b % 16, b // 16
    return x * f[..., 0].repeat_interleave(_GROUP, dim=-1) + f[..., 1].repeat_interleave(_GROUP, dim=-1)


def _turn64(x, pos, freqs, weight, order):
    """x [n, heads, hd] at positions pos [n], as complex numbers turned by pos * freq."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + _EPS) * weight.double()
    a = torch.outer(pos.double(), freqs.double())[:, None]
    z = torch.polar(torch.ones_like(a), a)
    half = x.shape[-1] // 2
    if order == "halves":
        y = torch.complex(x[..., :half], x[..., half:]) * z
        return torch.cat([y.real, y.imag], dim=-1)
    return torch.view_as_real(torch.view_as_complex(x.unflatten(-1, (half, 2)).contiguous()) * z).flatten(-2)


def _held64(x):
    """What the cache holds of rows x [..., hd] in 64 bits."""
    y = x.reshape(*x.shape[:-1], -1, _GROUP)
    m = y.min(-1, keepdim=True).values.half().double()
    s = ((y.max(-1, keepdim=True).values - y.min(-1, keepdim=True).values) / 15).half().double()
    return (torch.round((y - m) / s).clamp(0, 15) * s + m).reshape(x.shape)


def _exact_write(s):
    case = s["case"]
    stride, kvh, hd, new = (case[k] for k in ("stride", "kv_heads", "head_dim", "new"))
    out = {"q": [], "k": [], "k_cache": [], "v_cache": []}
    for b, (start, m) in enumerate(zip(_lengths(case), _new_lengths(case))):
        pos = start + torch.arange(new, device="cuda")
        out["q"].append(_turn64(s["q"][b], pos, s["freqs"], s["q_norm"], case["order"]))
        k = _turn64(s["k"][b], pos, s["freqs"], s["k_norm"], case["order"])
        out["k"].append(k)
        before = start % stride  # positions of the first page that are there already
        for slot, (name, x) in enumerate((("k_cache", k), ("v_cache", s["v"][b].double()))):
            got = torch.zeros(s["tail_ids"].shape[1] * stride, kvh, hd, dtype=torch.float64, device="cuda")
            got[:before] = _cached64(s, slot, s["tail_ids"][b].long())[:before]
            got[before:before + m] = _held64(x[:m])
            out[name].append(got)
    return {name: torch.stack(x) for name, x in out.items()}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "write":
        return _exact_write(s)
    if case["op"] == "prompt":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
        for b in range(case["bs"]):
            q, keys = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
            out[q] = _attend64(s["q"][q], s["k"][keys], s["v"][keys], case)
        return out
    lens = _lengths(case)
    width = s["ids"].shape[1] * case["stride"]
    cached = [[_cached64(s, slot, s["ids"][b].long())[:n] for slot in (0, 1)] for b, n in enumerate(lens)]
    if case["op"] == "read":
        fill = lambda x: torch.cat([x, x.new_zeros(width - x.shape[0], *x.shape[1:])])
        return {"k": torch.stack([fill(c[0]) for c in cached]), "v": torch.stack([fill(c[1]) for c in cached])}
    return torch.stack([_attend64(s["q"][b], *cached[b], case) for b in range(case["bs"])])
