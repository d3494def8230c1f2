"""The 8-bit KV cache as cases that can be timed and compared: writing it (with the
norms of queries and keys and the position rotation in the same pass), reading it
back, and attention over it.

  own         False: `run` computes the plain form; True: it calls the package
  listed()    the cases that stand for the range
  draw(rng)   one more case of the same range
  prepare     the activations, the page pool and the page table a serving loop holds
  run         one call, and what it gives
  work        bytes and flops one call cannot do without
  exact       what `run` gives, from the definition in 64 bits

Definitions.  A scale block is `scale_block` consecutive positions of a page; every
block, kv head and K | V has a scale s, and a code c stands for c * s.  A block whose
first position is written by a call gets s = amax / qmax (127, or 448 for e4m3) over the
rows written.  A block that is continued keeps its scale while the new rows fit (up to a
2^-10th part above qmax, which rounds back to qmax); otherwise its scale grows by the
smallest power of two that makes them fit and its earlier codes are rounded to the new
scale.
"""
from __future__ import annotations

import math

import torch

own = False

_BLOCKS, _BLOCK_INDEX = 2, 1  # transformer blocks in a page, the block called
_EPS = 1e-5
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_QMAX = {"int8": 127.0, "e4m3": 448.0}
_CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def _case(name, op, bs, positions, new=1, cache="int8", dtype="bf16", heads=32, kv_heads=8, head_dim=128, stride=32,
          scale_block=16, norm=False, order="pairs", softcap=0.0):
    """positions: cached positions of the longest sequence before the call (write) or in
    all (read, attend); new: new tokens of each sequence."""
    return {"name": name, "op": op, "bs": bs, "positions": positions, "new": new, "cache": cache, "dtype": dtype,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "stride": stride, "scale_block": scale_block,
            "norm": norm, "order": order, "softcap": softcap}


def listed():
    return [
        # one decode step of one sequence: launch latency
        _case("write_1x1_int8", "write", 1, 777),
        # a decode step of the largest batch, ragged positions inside their scale blocks
        _case("write_64x1_e4m3_norm", "write", 64, 4000, cache="e4m3", scale_block=32, norm=True),
        # one prompt of an odd length, half-split rotation, queries and keys normed
        _case("write_1x777_int8_norm_halves", "write", 1, 0, new=777, norm=True, order="halves"),
        # a batch of long prompts of the widest configuration
        _case("write_4x2048_e4m3", "write", 4, 0, new=2048, cache="e4m3", heads=48, scale_block=32),
        # the same pass over the framework's 16-bit cache
        _case("write_4x1024_bf16_norm", "write", 4, 0, new=1024, cache="bf16", norm=True),
        # the cached prefix of one short prompt, small heads
        _case("read_1x333_e4m3_f16", "read", 1, 333, cache="e4m3", dtype="f16", heads=16, kv_heads=4, head_dim=64,
              stride=16),
        # the cached prefixes of a full batch
        _case("read_32x4000_int8", "read", 32, 4000),
        # one decode step of one short sequence: launch latency
        _case("attend_1x100_int8", "attend", 1, 100),
        # the ordinary decode batch
        _case("attend_32x4000_int8", "attend", 32, 4000),
        # five drafted tokens of each sequence checked at once, the widest configuration with its softcap
        _case("attend_8x8190_new5_e4m3_cap", "attend", 8, 8190, new=5, cache="e4m3", heads=48, scale_block=32,
              softcap=30.0),
        # one sequence of a long context: the split over positions
        _case("attend_1x32768_int8", "attend", 1, 32768),
        # fp32 activations, small heads, a scale for each token
        _case("attend_16x1500_e4m3_f32", "attend", 16, 1500, cache="e4m3", dtype="f32", heads=16, kv_heads=4,
              head_dim=64, stride=16, scale_block=1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "write", "read", "attend", "attend", "attend"])
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (32, 8, 128), (48, 8, 128), (16, 4, 64), (8, 1, 128)])
    stride = rng.choice([16, 32, 32, 64])
    c = dict(cache=rng.choice(["int8", "e4m3"]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), heads=heads,
             kv_heads=kv_heads, head_dim=head_dim, stride=stride, scale_block=rng.choice([1, 4, 16, 16, stride]))
    bs = _log_int(rng, 1, 64)
    if op == "write":
        c.update(norm=rng.random() < 0.5, order=rng.choice(["pairs", "halves"]))
        if rng.random() < 0.2:
            c.update(cache=c["dtype"])
        if rng.random() < 0.5:  # a prompt batch
            new, positions = _log_int(rng, 2, 2048), rng.choice([0, 0, rng.randint(1, 2000)])
            bs = max(1, min(bs, 8192 // new))
        else:
            new, positions = 1, _log_int(rng, 16, 8192)
    elif op == "read":
        new, positions = 1, _log_int(rng, 16, 8192)
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
    """New tokens of each sequence: padded prompts are ragged, decode steps are not."""
    bs, n = case["bs"], case["new"]
    return [n - (i * (n // 3)) // bs for i in range(bs)] if n > 16 else [n] * bs


# ------------------------------------------------------------------------ inputs
def _scales_of(x, block, qmax):
    """x [..., positions, hd] -> the scale of each block, shaped [..., positions / block]."""
    return x.unflatten(-2, (-1, block)).abs().amax(dim=(-1, -2)) / qmax


def _codes_of(x, scale, block, cache):
    q = x.unflatten(-2, (-1, block)) / scale[..., None, None]
    q = q.clamp(-_QMAX[cache], _QMAX[cache])
    return (q.round() if cache == "int8" else q).to(_CODE[cache]).flatten(-3, -2)


def _freqs(hd):
    return (1.0 / (10000.0 ** (torch.arange(0, hd, 2).float() / hd))).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    bs, new, heads, kvh, hd, stride = (case[k] for k in ("bs", "new", "heads", "kv_heads", "head_dim", "stride"))
    dtype, eight = _DT[case["dtype"]], case["cache"] in _CODE
    lens = _lengths(case)
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    per_seq = -(-(case["positions"] + (new if case["op"] == "write" else 0)) // stride)
    pages = bs * per_seq + 1
    ids = (1 + torch.randperm(pages - 1, generator=gen, device="cuda")).view(bs, per_seq).to(torch.int32)
    s = {"case": case, "ids": ids, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    # the page pool; scores of standard deviation about 1.5
    if not eight:
        s["state"] = [torch.zeros(pages, _BLOCKS * 2 * stride * kvh * hd, dtype=dtype, device="cuda")]
    else:
        block = case["scale_block"]
        slab = torch.zeros(pages, _BLOCKS, kvh, 2, stride, hd, dtype=torch.int8, device="cuda").view(_CODE[case["cache"]])
        scales = torch.zeros(pages, _BLOCKS, kvh, stride // block, 2, device="cuda")
        if case["positions"]:
            x = rn(pages, kvh, 2, stride, hd) * 1.5
            sc = _scales_of(x, block, _QMAX[case["cache"]])
            slab.view(torch.int8)[:, _BLOCK_INDEX] = _codes_of(x, sc, block, case["cache"]).view(torch.int8)
            scales[:, _BLOCK_INDEX] = sc.transpose(-1, -2)
            del x, sc
        s["state"] = [slab.flatten(1), scales.flatten(1)]
    if case["op"] == "write":
        # one fused projection's output: q, k and v are views of it
        qkv = rn(bs, new, (heads + 2 * kvh) * hd).to(dtype)
        q, k, v = qkv.split([heads * hd, kvh * hd, kvh * hd], dim=-1)
        s["q"], s["k"], s["v"] = q.unflatten(-1, (heads, hd)), k.unflatten(-1, (kvh, hd)), v.unflatten(-1, (kvh, hd))
        s["freqs"] = _freqs(hd)
        s["q_norm"] = 1.0 + 0.1 * rn(hd) if case["norm"] else None
        s["k_norm"] = 1.0 + 0.1 * rn(hd) if case["norm"] else None
        news = _new_lengths(case)
        s["new_lens"] = torch.tensor(news, dtype=torch.int32, device="cuda") if new > 16 else None
        # the pages this call writes to, and how far they are filled after it
        first = [n // stride for n in lens]
        most = max((n + m - 1) // stride - f + 1 for n, m, f in zip(lens, news, first))
        at = torch.tensor(first, device="cuda")[:, None] + torch.arange(most, device="cuda")
        s["tail_ids"] = ids.gather(1, at.clamp(max=per_seq - 1))
        s["tail_lens"] = torch.tensor([n + m - f * stride for n, m, f in zip(lens, news, first)], dtype=torch.int32,
                                      device="cuda")
    elif case["op"] == "attend":
        s["q"] = rn(bs, new, heads, hd).to(dtype)
    if own:  # the handle of the package's cache, kept for the model's life
        from shark_platform_b200 import attention as A

        s["cache"] = A.PagedKVCache(transformer_block_count=_BLOCKS, attn_head_count=kvh, attn_head_dim=hd,
                                    block_seq_stride=stride, dtype=_CODE.get(case["cache"], dtype), device="cuda",
                                    scale_block=case["scale_block"] if eight else None)
    return s


# ------------------------------------------------------------------------ plain form
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
    slab = s["state"][0].unflatten(1, (_BLOCKS, case["kv_heads"], 2, case["stride"], case["head_dim"]))
    scales = s["state"][1].unflatten(1, (_BLOCKS, case["kv_heads"], case["stride"] // case["scale_block"], 2))
    return slab, scales


def _read(s, ids, lens):
    """Values of the listed pages, [bs, positions, kv_heads, hd] fp32 each, zero at and behind `lens`."""
    case = s["case"]
    slab, scales = _views(s)
    c = slab.view(torch.int8)[:, _BLOCK_INDEX][ids.long()].view(slab.dtype).float()  # [bs, n, heads, 2, stride, hd]
    sc = scales[:, _BLOCK_INDEX][ids.long()].transpose(-1, -2)                       # [bs, n, heads, 2, blocks]
    x = (c.unflatten(-2, (-1, case["scale_block"])) * sc[..., None, None]).flatten(-3, -2)
    x = x.permute(3, 0, 1, 4, 2, 5).flatten(2, 3)
    live = torch.arange(x.shape[2], device=x.device) < lens[:, None]
    return torch.where(live[None, :, :, None, None], x, torch.zeros((), device=x.device))


def _write8(s, kv):
    """kv [bs, new, kv_heads, 2, hd] fp32: quantised into the pages."""
    case = s["case"]
    block, stride, qmax = case["scale_block"], case["stride"], _QMAX[case["cache"]]
    slab, scales = _views(s)
    bs, new = kv.shape[:2]
    start = s["lens"].long()[:, None, None]
    count = new if s["new_lens"] is None else s["new_lens"].long()[:, None, None]
    slots = (new - 1) // block + (1 if new == 1 else 2)
    pos = (start // block + torch.arange(slots, device=kv.device)[None, :, None]) * block \
        + torch.arange(block, device=kv.device)                                     # [bs, slots, block]
    fresh, old = (pos >= start) & (pos < start + count), pos < start
    x = kv[torch.arange(bs, device=kv.device)[:, None, None], (pos - start).clamp(0, new - 1)]
    amax = torch.where(fresh[..., None, None, None], x.abs(), 0.0).amax(dim=(2, 5))  # [bs, slots, heads, 2]
    table = s["ids"].long().gather(1, (pos // stride).flatten(1).clamp(max=s["ids"].shape[1] - 1)).view_as(pos)
    at = (table[:, :, 0], torch.full_like(pos[:, :, 0], _BLOCK_INDEX))
    before = scales[at[0], at[1], :, pos[:, :, 0] % stride // block]                 # [bs, slots, heads, 2]
    s0 = torch.where(old[:, :, :1, None], before, 0.0)
    ratio = amax.double() / (s0.double() * qmax * (1 + 2.0 ** -10))
    grown = s0 * torch.exp2(torch.ceil(torch.log2(ratio.clamp(min=1.0)))).float()
    s1 = torch.where(s0 > 0, grown, amax / qmax)
    inv = torch.where(s1 > 0, 1.0 / s1.clamp(min=1e-37), 0.0)[:, :, None, :, :, None]
    shrink = torch.where(s1 > 0, s0 / s1.clamp(min=1e-37), 0.0)[:, :, None, :, :, None]  # a power of two, exact
    sel = table, torch.full_like(table, _BLOCK_INDEX), pos % stride
    held = slab.view(torch.int8)[sel[0], sel[1], :, :, sel[2]].view(slab.dtype).float()  # [bs, slots, block, heads, 2, hd]
    q = torch.where(fresh[..., None, None, None], x * inv, held * shrink).clamp(-qmax, qmax)
    codes = (q.round() if case["cache"] == "int8" else q).to(slab.dtype).view(torch.int8)
    live = (fresh | old) & fresh.any(-1, keepdim=True)
    slab.view(torch.int8)[sel[0][live], sel[1][live], :, :, sel[2][live]] = codes[live]
    some = fresh.any(-1)
    scales[at[0][some], _BLOCK_INDEX, :, (pos[:, :, 0] % stride // block)[some]] = s1[some]


def _write16(s, kv):
    """kv [bs, new, kv_heads, 2, hd] in the cache's type: into the pages."""
    case = s["case"]
    stride = case["stride"]
    slab = s["state"][0].unflatten(1, (_BLOCKS, 2, stride, case["kv_heads"], case["head_dim"]))
    bs, new = kv.shape[:2]
    i = torch.arange(new, device=kv.device)
    pos = s["lens"].long()[:, None] + i
    live = (i < (new if s["new_lens"] is None else s["new_lens"][:, None])).expand(bs, new)
    page = s["ids"].long().gather(1, pos // stride)
    slab[page[live], _BLOCK_INDEX, :, pos[live] % stride] = kv[live].transpose(1, 2)


def _plain_write(s):
    case = s["case"]
    dtype = _DT[case["dtype"]]
    pos = s["lens"].long()[:, None] + torch.arange(case["new"], device="cuda")
    q = _rotate(s["q"].float(), pos, s, s["q_norm"], case).to(dtype)
    k = _rotate(s["k"].float(), pos, s, s["k_norm"], case)
    kv = torch.stack([k, s["v"].float()], dim=3)
    if case["cache"] not in _CODE:
        _write16(s, kv.to(dtype))
        return {"q": q, "k": k.to(dtype), "cache": s["state"][0]}
    _write8(s, kv)
    kc, vc = _read(s, s["tail_ids"], s["tail_lens"]).to(dtype)
    return {"q": q, "k": k.to(dtype), "k_cache": kc, "v_cache": vc}


def _plain_attend(s):
    case = s["case"]
    k, v = _read(s, s["ids"], s["lens"])
    bs, new, heads, hd = s["q"].shape
    kvh = case["kv_heads"]
    q = s["q"].float().view(bs, new, kvh, heads // kvh, hd).permute(0, 2, 3, 1, 4).reshape(bs, kvh, -1, hd)
    w = torch.matmul(q, k.permute(0, 2, 3, 1)) * hd ** -0.5
    if case["softcap"]:
        w = case["softcap"] * torch.tanh(w / case["softcap"])
    w = w.view(bs, kvh, heads // kvh, new, -1)
    last = s["lens"][:, None] - new + torch.arange(new, device=w.device)
    dead = torch.arange(w.shape[-1], device=w.device) > last[..., None]
    w = w.masked_fill(dead[:, None, None], -math.inf)
    p = torch.exp(w - w.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v.transpose(1, 2)).view(bs, kvh, heads // kvh, new, hd)
    return o.permute(0, 3, 1, 2, 4).reshape(bs, new, heads, hd).to(s["q"].dtype)


# ------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    op, dtype = case["op"], _DT[case["dtype"]]
    if not own:
        if op == "write":
            return _plain_write(s)
        if op == "read":
            k, v = _read(s, s["ids"], s["lens"]).to(dtype)
            return {"k": k, "v": v}
        return _plain_attend(s)
    from shark_platform_b200 import attention as A

    cache, state = s["cache"], s["state"]
    if op == "write":
        q, k = A.norm_rope_kv_write(s["q"], s["k"], s["v"], cache, state, block_index=_BLOCK_INDEX,
                                    seq_block_ids=s["ids"], start_positions=s["lens"], new_lens=s["new_lens"],
                                    freqs=s["freqs"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=_EPS,
                                    use_hf=case["order"] == "halves")
        if case["cache"] not in _CODE:
            return {"q": q, "k": k, "cache": state[0]}
        # the values the written pages now stand for: what a continued prompt attends
        kc, vc = A.kv_read(cache, state, block_index=_BLOCK_INDEX, seq_block_ids=s["tail_ids"], seq_lens=s["tail_lens"],
                           dtype=dtype)
        return {"q": q, "k": k, "k_cache": kc, "v_cache": vc}
    if op == "read":
        k, v = A.kv_read(cache, state, block_index=_BLOCK_INDEX, seq_block_ids=s["ids"], seq_lens=s["lens"], dtype=dtype)
        return {"k": k, "v": v}
    return A.kv_attend(s["q"], cache, state, block_index=_BLOCK_INDEX, seq_block_ids=s["ids"], seq_lens=s["lens"],
                       softcap=case["softcap"] or None)


def work(case):
    bs, new, heads, kvh, hd, stride = (case[k] for k in ("bs", "new", "heads", "kv_heads", "head_dim", "stride"))
    io = 4 if case["dtype"] == "f32" else 2
    lens, block = _lengths(case), case["scale_block"]
    held = lambda n: kvh * (2 * n * hd + 8 * -(-n // block))  # codes and scales of n positions
    if case["op"] == "write":
        news = _new_lengths(case)
        bytes_ = bs * new * hd * io * (2 * heads + 3 * kvh)  # q, k, v read; q and k written (padding rows too)
        if case["cache"] in _CODE:
            # written, and the filled part of the written pages read back into rows of the activations' type
            tail = [n % stride + m for n, m in zip(lens, news)]
            rows = bs * max(-(-t // stride) for t in tail) * stride
            bytes_ += sum(held(m) for m in news) + sum(held(t) for t in tail) + rows * 2 * kvh * hd * io
        else:
            bytes_ += sum(news) * 2 * kvh * hd * io
        return {"bytes": bytes_, "flops": bs * new * (heads + kvh) * hd * 8}
    if case["op"] == "read":
        rows = bs * -(-case["positions"] // stride) * stride
        return {"bytes": sum(held(n) for n in lens) + rows * 2 * kvh * hd * io, "flops": 2 * sum(lens) * kvh * hd}
    attended = sum(n - new + 1 + i for n in lens for i in range(new))
    return {"bytes": sum(held(n) for n in lens) + 2 * bs * new * heads * hd * io, "flops": 4 * attended * heads * hd}


# ------------------------------------------------------------------------ 64 bits
def _code64(y, cache):
    """Codes for y = value / scale, in 64 bits; e4m3: 3 bits behind the leading one, steps of 2^-9 below 2^-6."""
    y = y.clamp(-_QMAX[cache], _QMAX[cache])
    if cache == "int8":
        return torch.round(y)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def _cached64(s, slot, pages):
    """K (slot 0) or V (1) of a list of pages, [positions, kv_heads, hd]; and codes and scales as they are held."""
    case = s["case"]
    slab, scales = _views(s)
    c = slab.view(torch.int8)[pages, _BLOCK_INDEX, :, slot].view(slab.dtype).double()   # [n, heads, stride, hd]
    f = scales[pages, _BLOCK_INDEX, :, :, slot].double()                                # [n, heads, blocks]
    c, f = c.transpose(1, 2).flatten(0, 1), f.transpose(1, 2).flatten(0, 1)             # positions / blocks first
    return c * f.repeat_interleave(case["scale_block"], dim=0)[..., None], c, f


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


def _exact_write(s):
    case = s["case"]
    stride, block, hd, kvh, new = (case[k] for k in ("stride", "scale_block", "head_dim", "kv_heads", "new"))
    eight, news, lens = case["cache"] in _CODE, _new_lengths(case), _lengths(case)
    out_q, out_k, kv_out = [], [], []
    cache = None if eight else s["state"][0].double().view(-1, _BLOCKS, 2, stride, kvh, hd).clone()
    width = s["tail_ids"].shape[1] * stride
    for b, (start, m) in enumerate(zip(lens, news)):
        pos = start + torch.arange(new, device="cuda")
        out_q.append(_turn64(s["q"][b], pos, s["freqs"], s["q_norm"], case["order"]))
        k = _turn64(s["k"][b], pos, s["freqs"], s["k_norm"], case["order"])
        out_k.append(k)
        pair = []
        base = start // stride * stride  # first position of the pages that are read back
        for slot, x in enumerate((k, s["v"][b].double())):
            if not eight:
                at = pos[:m]
                cache[s["ids"][b].long()[at // stride], _BLOCK_INDEX, slot, at % stride] = x[:m]
                continue
            val, c, f = _cached64(s, slot, s["tail_ids"][b].long())
            got = torch.zeros(width, kvh, hd, dtype=torch.float64, device="cuda")
            got[:start - base] = val[:start - base]
            # the block that is continued, then the whole fresh ones at once
            cut = min(m, -start % block)
            qmax = _QMAX[case["cache"]]
            if cut:
                lo = start // block * block - base
                s0, top = f[lo // block], x[:cut].abs().amax(dim=(0, 2))
                grow = torch.ceil(torch.log2((top / (s0 * qmax * (1 + 2.0 ** -10))).clamp(min=1.0)))
                s1 = s0 * torch.exp2(grow)
                old = _code64(c[lo:start - base] * torch.exp2(-grow)[:, None], case["cache"])
                got[lo:start - base] = old * s1[:, None]
                got[start - base:start - base + cut] = _code64(x[:cut] / s1[:, None], case["cache"]) * s1[:, None]
            if m > cut:
                rest = x[cut:m]
                pad = -rest.shape[0] % block
                y = torch.cat([rest, rest.new_zeros(pad, kvh, hd)]).unflatten(0, (-1, block))
                sc = y.abs().amax(dim=(1, 3), keepdim=True) / qmax
                y = (_code64(y / sc, case["cache"]) * sc).flatten(0, 1)[:m - cut]
                got[start - base + cut:start - base + m] = y
            pair.append(got)
        kv_out.append(pair)
    res = {"q": torch.stack(out_q), "k": torch.stack(out_k)}
    if not eight:
        return {**res, "cache": cache.flatten(1)}
    return {**res, "k_cache": torch.stack([p[0] for p in kv_out]), "v_cache": torch.stack([p[1] for p in kv_out])}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "write":
        return _exact_write(s)
    outs = []
    width = s["ids"].shape[1] * case["stride"]
    group = case["heads"] // case["kv_heads"]
    for b, n in enumerate(_lengths(case)):
        k, v = (_cached64(s, slot, s["ids"][b].long())[0][:n] for slot in (0, 1))
        if case["op"] == "read":
            outs.append([torch.cat([x, x.new_zeros(width - n, *x.shape[1:])]) for x in (k, v)])
            continue
        rows = []
        for i in range(case["new"]):
            m = n - case["new"] + 1 + i
            q = s["q"][b, i].double().view(case["kv_heads"], group, -1)
            w = torch.einsum("hgd,nhd->hgn", q, k[:m]) / math.sqrt(case["head_dim"])
            if case["softcap"]:
                w = torch.tanh(w / case["softcap"]) * case["softcap"]
            rows.append(torch.einsum("hgn,nhd->hgd", torch.softmax(w, dim=-1), v[:m]).flatten(0, 1))
        outs.append(torch.stack(rows))
    if case["op"] == "read":
        return {"k": torch.stack([o[0] for o in outs]), "v": torch.stack([o[1] for o in outs])}
    return torch.stack(outs)
