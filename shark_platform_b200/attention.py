"""The attention block that precedes every MoE layer, on the GPU.

`B200PagedAttentionBlock` has the constructor and `forward` of sharktank's
`PagedLlamaAttentionBlock` (layers/paged_llama_attention_block.py:26-303) and
works on the same objects: the model's theta (`attn_norm`, `attn_q`, `attn_k`,
`attn_v`, `attn_output`, optional `attn_output_norm`), a `PagedKVCache`
(layers/kv_cache.py:222-526; sharktank's own or the mirror below), the list
`cache_state` holding the page slab, and a rotary embedding layer.

With a cache of 8-bit codes (`PagedKVCache(dtype=torch.int8 | torch.float8_e4m3fn)`),
per-head query / key norms (`attn_q_norm`, `attn_k_norm` in the theta), the HuggingFace
rotation order or `new_lens`, the block takes the operators below instead of the rotary
kernel; they are public on their own:
  * `norm_rope_kv_write`: norms, rotation and the (quantising) cache write in one pass;
  * `kv_attend`: attention of one or a few new tokens over an 8-bit cache;
  * `kv_read`: the values of an 8-bit cache as plain K and V.
All of them take caches of 4-bit codes as well (`PagedKVCache(dtype=torch.uint8)`).
`prompt_attend` is the attention of whole prompts: packed sequences, causal, grouped heads.

What runs where:
  * RMS norm, rotary embedding fused with the KV page write, and the decode
    attention over the pages: this library's kernels (`b200moe_rms_norm`,
    `b200moe_attn_rope_kv_write`, `b200moe_attn_decode`).  Decode never
    materialises the linear K/V temporaries the reference reads the cache into
    (`xk_temp` / `xv_temp` are accepted and ignored).
  * the four projections: one dense product each (q, k and v fused into one) —
    a library GEMM for dense weights, this library's quantized linear for Q8_0 /
    Q4_K / Q4_1 weights;
  * the prefill attention core over the freshly computed K/V: with
    `attention_kernel="b200"` this library's `prompt_attend`, as with a cache of 4-bit
    codes and no mask; else torch's fused scaled-dot-product attention, which the
    reference also offers as `attention_kernel="torch"` (:215-224); with a softcap (Grok)
    the decomposed torch operators, since the fused kernel has no cap.

There is no CPU path: CPU tensors are rejected.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch
import torch.nn.functional as F

from . import _cabi as C
from . import moe as _moe

_DT = {torch.float32: C.DT_F32, torch.float16: C.DT_F16, torch.bfloat16: C.DT_BF16}


def _p(t: Optional[torch.Tensor]):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


_CODES = {torch.int8: C.KV8_INT8, torch.float8_e4m3fn: C.KV8_E4M3, torch.uint8: C.KV4}
KV4_GROUP = 32       # values of a row that share a scale and an offset, 4-bit codes
MAX_NEW_TOKENS = 16  # of one kv_attend call


class PagedKVCache:
    """Mirror of sharktank's PagedKVCache (layers/kv_cache.py:222-340) for use
    without sharktank: geometry plus `allocate`.  Reads and writes happen inside
    the attention block's kernels.

    `dtype` int8 or float8_e4m3fn makes it a cache of 8-bit codes with one fp32
    scale for each `scale_block` consecutive positions of a page, kv head and K | V
    (a power of two up to 64 that divides `block_seq_stride`; by default the largest
    one up to 16): 1 + 4 / scale_block / head_dim bytes per value.  Small blocks follow
    single large rows more closely, large ones have fewer scales to read.

    `dtype` uint8 makes it a cache of 4-bit codes, two a byte, with an fp16 scale and offset
    for each 32 values of a row: 5 / 8 bytes per value.  Rows are independent of each other."""

    def __init__(self, *, transformer_block_count: int, attn_head_count: int, attn_head_dim: int,
                 cache_partition_count: int = 2, block_seq_stride: int = 16,
                 dtype: torch.dtype = torch.float32, device=None, shard_count: int = 1,
                 scale_block: Optional[int] = None):
        if cache_partition_count != 2 or shard_count != 1:
            raise C.B200MoeError("the cache holds K and V on one device")
        self.transformer_block_count = transformer_block_count
        self.attn_head_count = attn_head_count
        self.attn_head_dim = attn_head_dim
        self.cache_partition_count = cache_partition_count
        self.block_seq_stride = block_seq_stride
        self.shard_count = shard_count
        self.dtype, self.device = dtype, device
        self.quantized = dtype in _CODES
        self.scale_dtype = None
        if dtype == torch.uint8:
            if scale_block is not None:
                raise C.B200MoeError("scale_block is for caches of 8-bit codes, not 4-bit ones")
            if attn_head_dim % KV4_GROUP:
                raise C.B200MoeError(f"head_dim {attn_head_dim}: a cache of 4-bit codes has scales for {KV4_GROUP} values each")
            self.scale_block = None
            self.scale_dtype = torch.float16
            # a head's rows of a page are one contiguous stretch; scales and offsets: the same rows
            self.sub_page_dims = [transformer_block_count, attn_head_count, 2, block_seq_stride, attn_head_dim // 2]
            self.scale_page_dims = [transformer_block_count, attn_head_count, 2, block_seq_stride, attn_head_dim // KV4_GROUP, 2]
            self.scale_flat_dim = math.prod(self.scale_page_dims)
        elif self.quantized:
            self.scale_dtype = torch.float32
            # the largest power of two that divides the stride, up to 16
            self.scale_block = min(block_seq_stride & -block_seq_stride, 16) if scale_block is None else scale_block
            b = self.scale_block
            if b < 1 or b > 64 or b & (b - 1) or block_seq_stride % b:
                raise C.B200MoeError(f"scale_block {b}: a power of two up to 64 that divides the page stride "
                                     f"({block_seq_stride})")
            # a page's rows of one head are one contiguous stretch
            self.sub_page_dims = [transformer_block_count, attn_head_count, 2, block_seq_stride, attn_head_dim]
            self.scale_page_dims = [transformer_block_count, attn_head_count, block_seq_stride // b, 2]
            self.scale_flat_dim = math.prod(self.scale_page_dims)
        else:
            if scale_block is not None:
                raise C.B200MoeError(f"scale_block is for caches of 8-bit codes, not {dtype}")
            self.scale_block = None
            self.sub_page_dims = [transformer_block_count, 2, block_seq_stride, attn_head_count, attn_head_dim]
        self.page_slab_flat_dim = math.prod(self.sub_page_dims)
        self._geometry = (transformer_block_count, block_seq_stride, attn_head_count, attn_head_dim,
                          self.scale_block or 1, _CODES.get(dtype, -1))

    def allocate(self, page_count: int) -> list[torch.Tensor]:
        """[page slab], or [page slab, scales] for 8- and 4-bit codes: a row of each per page."""
        state = [torch.zeros(page_count, self.page_slab_flat_dim, dtype=self.dtype, device=self.device)]
        if self.quantized:
            state.append(torch.zeros(page_count, self.scale_flat_dim, dtype=self.scale_dtype, device=self.device))
        return state


# ------------------------------------------------------------- cache operators
# Checks, outputs and launches are in csrc/attention_ops.cpp: these are called once per layer
# and token.
def _geometry(cache) -> tuple:
    g = getattr(cache, "_geometry", None)  # sharktank's own PagedKVCache: 16- or 32-bit
    return g if g is not None else (cache.transformer_block_count, cache.block_seq_stride, cache.attn_head_count,
                                    cache.attn_head_dim, 1, -1)


def norm_rope_kv_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: PagedKVCache, cache_state: list, *,
                       block_index: int, seq_block_ids: torch.Tensor, start_positions: torch.Tensor,
                       freqs: torch.Tensor, new_lens: Optional[torch.Tensor] = None,
                       q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                       eps: float = 1e-5, use_hf: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Puts new tokens into the cache: RMS norm of every query and key head (`q_norm`,
    `k_norm`: fp32 [head_dim], or None), rotation by position * `freqs` (fp32
    [head_dim / 2]; pairs (2i, 2i + 1), with `use_hf` (i, i + head_dim / 2)), and K and V
    written to their pages, quantised if the cache holds 8-bit codes: one pass.

    q [bs, sl, heads, head_dim], k and v [bs, sl, kv_heads, head_dim] (views of one fused
    projection are taken as they are) hold tokens start_positions[b] ... + sl - 1 of
    sequence b; those at and behind new_lens[b] are padding: rotated, not written.  A
    negative start position makes a whole sequence padding.  Sequences of one call must
    not share the pages they write.  Returns the rotated q and k, contiguous.

    8-bit codes: a scale block that the call begins has the scale amax / 127 (448 for
    e4m3) of the rows written; one that it continues keeps its scale while the new rows
    fit, else the scale grows by a power of two and the block's earlier codes are rounded
    to it.  Positions behind the last written one of a block are dead until written (a
    drafted token that is taken back leaves its block's scale as it made it).  An infinity
    or NaN makes its block read as NaN until it is begun again.

    4-bit codes: every 32 values of a row have the scale (max - min) / 15 and the offset min,
    rounded to fp16, and the codes nearest to them.  Rows are independent: any position may be
    written again at any time.  A group with an infinity or a NaN, or whose scale or offset
    is beyond fp16's range, reads as NaN: in `kv_attend` a group of K makes the whole output of
    the rows that see it NaN, one of V its own 32 elements."""
    return C.attention_ops.write(q, k, v, cache_state, _geometry(cache), block_index, seq_block_ids, start_positions, new_lens,
                                 freqs, q_norm, k_norm, eps, use_hf)


def kv_read(cache: PagedKVCache, cache_state: list, *, block_index: int, seq_block_ids: torch.Tensor,
            seq_lens: torch.Tensor, max_seq_len: Optional[int] = None,
            dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of the listed pages of an 8- or 4-bit cache, [bs, max_seq_len, kv_heads, head_dim]
    each (`max_seq_len`: all of the listed pages by default); every value code * scale
    (+ offset), rounded once to `dtype`.  Rows at and behind seq_lens[b] are zero."""
    return C.attention_ops.read(cache_state, _geometry(cache), block_index, seq_block_ids, seq_lens, max_seq_len, dtype)


def kv_attend(q: torch.Tensor, cache: PagedKVCache, cache_state: list, *, block_index: int,
              seq_block_ids: torch.Tensor, seq_lens: torch.Tensor, scale: Optional[float] = None,
              softcap: Optional[float] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Attention of the last sl (1 ... 16) positions of each sequence over an 8- or 4-bit cache.

    q [bs, sl, heads, head_dim], rotated; seq_lens[b] counts the positions in the cache,
    the sl new ones included (`norm_rope_kv_write` first).  Token i attends the positions
    up to and including its own, seq_lens[b] - sl + i; where that leaves none its output is
    zero.  scale: 1 / sqrt(head_dim) by default; softcap: c * tanh(score / c).  Returns
    [bs, sl, heads, head_dim].

    Sums and softmax statistics are 32-bit.  The probabilities are rounded to 22 bits where the
    output is fp32 or fp16 or q is fp32, else (bf16) to 11, an eighth of the output's rounding."""
    return C.attention_ops.attend(q, cache_state, _geometry(cache), block_index, seq_block_ids, seq_lens, scale, softcap,
                                  out_dtype)


def prompt_attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, cu_seqlens: torch.Tensor,
                  cu_seqlens_k: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                  softcap: Optional[float] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Causal attention of packed sequences of different lengths, without padding.

    q [rows, heads, head_dim], k and v [rows, kv_heads, head_dim], rotated (views of one fused
    projection are taken as they are).  Sequence b has q's rows cu_seqlens[b] ...
    cu_seqlens[b + 1] - 1 (whole numbers on q's device, bs + 1 of them) and the rows of k and v
    that cu_seqlens_k says, by default the same.  A continued prompt has more rows of k than of
    q, its last ones being those of q: of n rows of q and m of k, row i attends rows 0 ...
    m - n + i.  Where that leaves none the output is zero, as it is for rows of no sequence
    (in front of the first and behind the last).  scale: 1 / sqrt(head_dim) by default; softcap:
    c * tanh(score / c).  Returns [rows, heads, head_dim] of `out_dtype`, by default q's.

    An infinity or NaN in v shows in the rows that attend it, and only there: as an infinity, or as
    NaN where its weight is zero in the products' type.  Sums and softmax statistics are 32-bit;
    the weights of 16-bit rows are rounded to their type, also where the output is of 32 bits.
    There is no gradient: inputs that want one are refused."""
    return C.attention_ops.prompt(q, k, v, cu_seqlens, cu_seqlens_k, scale, softcap, out_dtype)


class RotaryEmbeddingLayer:
    """What the block needs of sharktank's RotaryEmbeddingLayer
    (layers/rotary_embedding.py:20-40): the dimension count and the frequency base."""

    def __init__(self, *, rope_dimension_count: int, max_seqlen: int, rope_freq_base: Optional[float] = None,
                 device=None, use_hf: bool = False):
        self.rope_dimension_count = rope_dimension_count
        self.max_seqlen = max_seqlen
        self.rope_freq_base = rope_freq_base if rope_freq_base is not None else 10000.0
        self.device, self.use_hf = device, use_hf


def _is_quantized(t) -> bool:
    return _moe._layout_name(t) in _moe._SUPPORTED


def _check_causal(mask: torch.Tensor, bs: int, new_lens: Optional[torch.Tensor], device) -> None:
    """Sets the status word's bounds bit where a row of tokens of `mask` [..., sl, sl or more] sees
    other positions than the causal ones.  A position is seen where the mask is zero (True, for truth
    values) and not where it is -5000 or less; anything else is no mask.  The tokens of a sequence are
    the rows that see their own position, and those that new_lens says."""
    if mask.dtype == torch.bool:
        mask = torch.zeros(mask.shape, device=mask.device).masked_fill_(~mask, float("-inf"))
    mask = mask.to(device, mask.dtype if mask.dtype in _DT else torch.float32)
    for d in range(mask.dim() - 2):  # expanded dimensions once
        if mask.stride(d) == 0:
            mask = mask.narrow(d, 0, 1)
    own = mask.dim() == 4 and mask.shape[0] == bs  # each sequence has its own
    per = mask.shape[1] if own else 0
    mask = mask.reshape(-1, *mask.shape[-2:])
    if mask.stride(2) != 1:
        mask = mask.contiguous()
    lens = None if new_lens is None else new_lens.to(device, torch.int32).contiguous()
    with torch.cuda.device(device):
        C.check(C.lib.b200moe_causal_mask_check(_p(mask), _DT[mask.dtype], mask.stride(0), mask.stride(1), *mask.shape, _p(lens), bs, per,
                                                _moe._stream()), "causal_mask_check")


class B200PagedAttentionBlock(torch.nn.Module):
    """Drop-in for PagedLlamaAttentionBlock (same constructor keywords, same
    `forward` keywords).

    `attention_kernel="b200"` takes `prompt_attend` for prompts.  It is causal by itself: an
    `attention_mask` has to be the causal one, with any padding behind a sequence's tokens (the
    rows of padding are attended too and mean nothing).  One whose shape cannot be that is
    refused; its values are looked at on the device: where a row of tokens sees other
    positions the status word's bounds bit is set (`moe.device_status` raises)."""

    def __init__(self, theta, *, block_index: int, cache, head_count: int, head_dim: int, head_count_kv: int,
                 rms_epsilon: float, attention_kernel: str = "decomposed", attention_scale: Optional[float] = None,
                 softcap: Optional[float] = None, fake_quant: Optional[bool] = True):
        super().__init__()
        self.theta = theta
        self.block_index, self.cache = block_index, cache
        self.head_count, self.head_dim, self.head_count_kv = head_count, head_dim, head_count_kv
        self.rms_epsilon = rms_epsilon
        self.attention_kernel, self.attention_scale, self.softcap = attention_kernel, attention_scale, softcap
        if "kv_cache" in getattr(theta, "keys", ()):
            raise C.B200MoeError("a quantized KV cache (kv_cache.quantizer) is not supported: its one scale per tensor "
                                 "is replaced by PagedKVCache(dtype=torch.int8, torch.float8_e4m3fn or torch.uint8)")
        self._quantized = bool(getattr(cache, "quantized", False))
        if head_count % head_count_kv != 0 or (head_count // head_count_kv > 8 and not self._quantized):
            raise C.B200MoeError("head_count must be 1..8 times head_count_kv (any multiple with an 8- or 4-bit cache)")
        if head_dim not in (64, 128):
            raise C.B200MoeError(f"head_dim {head_dim}: 64 and 128 are built")
        if cache.attn_head_count != head_count_kv or cache.attn_head_dim != head_dim:
            raise C.B200MoeError("the cache's heads / head_dim differ from the block's")
        w = lambda name: theta(name).tensor("weight")
        self._norm_w = _moe._aligned(_moe._unbox(w("attn_norm")).to(torch.float32))
        _moe._require_cuda(self._norm_w, "attn_norm.weight")
        self._out_norm_w = None
        if theta.optional_tensor("attn_output_norm") is not None:
            self._out_norm_w = _moe._unbox(w("attn_output_norm")).to(torch.float32).contiguous()
        # norms of every query and key head, before the rotation
        self._q_norm_w, self._k_norm_w = (
            _moe._unbox(w(n)).to(torch.float32).contiguous() if n in theta.keys else None
            for n in ("attn_q_norm", "attn_k_norm"))
        for x in (self._q_norm_w, self._k_norm_w):
            if x is not None and x.shape != (head_dim,):
                raise C.B200MoeError(f"attn_q_norm and attn_k_norm have one weight per element of a head ({head_dim})")
        wq, wk, wv, self._wo = w("attn_q"), w("attn_k"), w("attn_v"), w("attn_output")
        self._bias = {n: theta(n).optional_tensor("bias") if "bias" in theta(n).keys else None
                      for n in ("attn_q", "attn_k", "attn_v", "attn_output")}
        if any(_is_quantized(t) for t in (wq, wk, wv)):
            self._wqkv, self._wq, self._wk, self._wv = None, wq, wk, wv
        else:  # one fused projection
            self._wqkv = torch.cat([_moe._unbox(t) for t in (wq, wk, wv)], dim=0).contiguous()
        self._freqs = None
        self._desc = C.KvCacheDesc(cache.transformer_block_count, cache.block_seq_stride, head_count_kv, head_dim, 0)

    # ---------------------------------------------------------------- pieces
    def _linear(self, x, weight, bias):
        if _is_quantized(weight):
            y = _moe.linear_quantized(x, weight, bias)
            if y is NotImplemented:
                raise C.B200MoeError("quantized projection weight has an unsupported shape")
            return y
        wt = _moe._unbox(weight) if not isinstance(weight, torch.Tensor) else weight
        return F.linear(x, wt.to(x.dtype), None if bias is None else _moe._unbox(bias).to(x.dtype))

    @staticmethod
    def _fits_linear(*weights) -> bool:
        """Every weight is one that `moe.matmul_quantized` takes."""
        return all(_is_quantized(w) and len(w.shape) == 2 and int(w.shape[0]) % 256 == 0 and
                   int(w.shape[1]) % 256 == 0 for w in weights)

    def _norm(self, x, weight):
        y = torch.empty_like(x)
        rows = x.numel() // x.shape[-1]
        with torch.cuda.device(x.device):
            C.check(C.lib.b200moe_rms_norm(_p(x), _DT[x.dtype], _p(weight), rows, x.shape[-1],
                                           float(self.rms_epsilon), _p(y), _DT[y.dtype], _moe._stream()), "rms_norm")
        return y

    def _freq_table(self, embedding, device):
        if self._freqs is None or self._freqs.device != device:
            dim = embedding.rope_dimension_count
            if dim != self.head_dim:
                raise C.B200MoeError("rope_dimension_count must equal head_dim")
            base = embedding.rope_freq_base
            # layers/rotary_embedding.py:222-228, one entry per pair
            freqs = 1.0 / (base ** ((torch.arange(0, dim) // 2).float() / dim * 2.0))
            self._freqs = freqs[0::2].contiguous().to(device)
        return self._freqs

    def _torch_attention(self, q, k, v, attention_mask, before, scale):
        """Prefill by torch's operators: q [bs, sl, heads, hd], k and v [bs, before + sl, kv_heads, hd]."""
        bs, sl, H, hd = q.shape
        Hkv = k.shape[2]
        qh, kh, vh = q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)
        mask = None if attention_mask is None else attention_mask.to(q.dtype)
        if before:
            if mask is None:
                mask = torch.full((sl, before + sl), float("-inf"), device=q.device, dtype=q.dtype).triu(before + 1)
            elif mask.shape[-1] == sl:
                mask = F.pad(mask, (before, 0))
        if self.softcap is None:
            attn = F.scaled_dot_product_attention(qh, kh, vh, attn_mask=mask, is_causal=mask is None, scale=scale,
                                                  enable_gqa=H != Hkv)
        else:
            rep = H // Hkv
            kh, vh = kh.repeat_interleave(rep, dim=1), vh.repeat_interleave(rep, dim=1)
            w = torch.matmul(qh, kh.transpose(2, 3)) * scale
            w = self.softcap * torch.tanh(w / self.softcap)
            if mask is not None:
                w = w + mask
            else:
                w = w + torch.full((sl, sl), float("-inf"), device=q.device, dtype=w.dtype).triu(1)
            attn = torch.matmul(torch.softmax(w.float(), dim=-1).to(qh.dtype), vh)
        return attn.transpose(1, 2)

    # --------------------------------------------------------------- forward
    def forward(self, h: torch.Tensor, *, embedding, seq_block_ids: torch.Tensor,
                start_index: Optional[int] = None, start_positions: Optional[torch.Tensor] = None,
                attention_mask: Optional[torch.Tensor] = None, embedding_batch_mask: Optional[torch.Tensor] = None,
                cache_state: list = None, xk_temp: Optional[torch.Tensor] = None,
                xv_temp: Optional[torch.Tensor] = None, new_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """`new_lens` [bs] (prefill; not in the reference): how many of each sequence's rows are
        tokens; padding behind them is not written to the cache.  With an 8- or 4-bit cache a decode
        step may bring up to 16 tokens per sequence (each attends the ones before it), a
        negative start position marks a padding sequence, and a prefill with start_index > 0
        attends the cached positions before it too (an attention_mask then covers the new
        positions, or all of them).  With a 16- or 32-bit cache a prefill attends its new positions
        only, as the reference's does; with norms, the HuggingFace order or `new_lens` such a
        call with start_index > 0 is refused."""
        _moe._require_cuda(h, "h")
        if h.dtype not in _DT:
            raise C.B200MoeError(f"activations must be fp32, fp16 or bf16, got {h.dtype}")
        if (start_index is not None) == (start_positions is not None):
            raise C.B200MoeError("exactly one of start_index (prefill) and start_positions (decode) is given")
        slab = cache_state[0]
        if not self._quantized and (slab.dtype not in _DT or not slab.is_contiguous()):
            raise C.B200MoeError("the page slab must be a contiguous fp32, fp16 or bf16 tensor")
        dev = h.device
        bs, sl, d = h.shape
        H, Hkv, hd = self.head_count, self.head_count_kv, self.head_dim
        stride = self.cache.block_seq_stride
        decode = start_positions is not None
        if decode and sl != 1 and not self._quantized:
            raise C.B200MoeError("a decode step brings one token per sequence")
        if decode and sl > MAX_NEW_TOKENS:
            raise C.B200MoeError(f"a decode step brings at most {MAX_NEW_TOKENS} tokens per sequence")
        if decode and new_lens is not None:
            raise C.B200MoeError("new_lens is for prefill; a negative start position marks a padding sequence of a step")
        if not decode and self.attention_kernel == "b200" and attention_mask is not None:
            seen = {sl, int(start_index) + sl} if self._quantized else {sl}
            lead = attention_mask.shape[:-2]
            if (not 2 <= attention_mask.dim() <= 4 or attention_mask.shape[-2] != sl or attention_mask.shape[-1] not in seen or
                    any(n not in (1, most) for n, most in zip(reversed(lead), (H, bs)))):
                raise C.B200MoeError('attention_kernel="b200" is causal by itself: an attention_mask of '
                                     f"{list(attention_mask.shape)} is not the causal one of {sl} tokens")
        use_hf = bool(getattr(embedding, "use_hf", False))
        # norms, the HuggingFace order, padding and 8-bit codes: the one-pass write
        one_pass = (self._quantized or use_hf or new_lens is not None or self._q_norm_w is not None or
                    self._k_norm_w is not None)
        if one_pass and not decode and (int(start_index) < 0 or (int(start_index) > 0 and not self._quantized)):
            raise C.B200MoeError(f"a prefill from position {int(start_index)}: continued prompts are for 8- and 4-bit caches "
                                 "(the positions before it would not be attended)")
        hc = h.contiguous()
        # the output projection with the residual, in one call
        fused_out = (self._fits_linear(self._wo) and [int(n) for n in self._wo.shape] == [d, H * hd] and
                     self._bias["attn_output"] is None and self._out_norm_w is None)
        if self._wqkv is not None:
            x = self._norm(hc, self._norm_w)
            qkv = F.linear(x, self._wqkv.to(x.dtype))
            q, k, v = torch.split(qkv, [H * hd, Hkv * hd, Hkv * hd], dim=-1)
            if not one_pass:
                q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        elif self._fits_linear(self._wq, self._wk, self._wv) and int(self._wq.shape[1]) == d:
            # norm and the three projections in one call
            q, k, v = _moe.linear_rows(hc.view(bs * sl, d), [_moe.prepare_linear(w) for w in (self._wq, self._wk, self._wv)],
                                       norm_weight=self._norm_w, eps=float(self.rms_epsilon))
            q, k, v = (y if bias is None else y + _moe._unbox(bias).to(y.dtype) for y, bias in
                       zip((q, k, v), (self._bias[n] for n in ("attn_q", "attn_k", "attn_v"))))
        else:
            x = self._norm(hc, self._norm_w)
            q = self._linear(x, self._wq, self._bias["attn_q"]).contiguous()
            k = self._linear(x, self._wk, self._bias["attn_k"]).contiguous()
            v = self._linear(x, self._wv, self._bias["attn_v"]).contiguous()
        if self._wqkv is not None and any(self._bias[n] is not None for n in ("attn_q", "attn_k", "attn_v")):
            raise C.B200MoeError("projection biases are supported with unfused (quantized) weights only")
        own = not decode and (self.attention_kernel == "b200" or
                              (getattr(self.cache, "dtype", None) == torch.uint8 and attention_mask is None))
        if own and torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v)):
            raise C.B200MoeError("the packed prompt attention has no gradient: call the block under torch.no_grad()")
        tokens = bs * sl
        page_ids = seq_block_ids.to(torch.int32).contiguous()
        self._desc.page_count = slab.shape[0]
        if one_pass:
            start = (start_positions.to(torch.int32).contiguous() if decode else
                     torch.full((bs,), int(start_index), device=dev, dtype=torch.int32))
            q, k = norm_rope_kv_write(q.view(bs, sl, H, hd), k.view(bs, sl, Hkv, hd), v.view(bs, sl, Hkv, hd), self.cache,
                                      cache_state, block_index=self.block_index, seq_block_ids=page_ids,
                                      start_positions=start, new_lens=new_lens, freqs=self._freq_table(embedding, dev),
                                      q_norm=self._q_norm_w, k_norm=self._k_norm_w, eps=float(self.rms_epsilon),
                                      use_hf=use_hf)
            positions = start
        else:
            if decode:
                positions = start_positions.to(torch.int32).contiguous()
            else:
                positions = (torch.arange(sl, device=dev, dtype=torch.int32) + int(start_index)).repeat(bs)
            # prefill attends the fresh K and V: K is rotated in place, V is used as it is
            k_out, v_out = (None, None) if decode else (k, v)
            with torch.cuda.device(dev):
                C.check(C.lib.b200moe_attn_rope_kv_write(
                    _p(q), _p(k), _p(v), _p(k_out), _p(v_out), _DT[q.dtype], _p(slab), _DT[slab.dtype],
                    ctypes.byref(self._desc), self.block_index, _p(positions), _p(page_ids),
                    _p(self._freq_table(embedding, dev)), tokens, sl, page_ids.shape[1], H, _moe._stream()),
                    "attn_rope_kv_write")
        scale = self.attention_scale if self.attention_scale is not None else 1.0 / math.sqrt(hd)
        # a Q8_0 output projection reads fp16 rows: no cast in between
        direct = fused_out and _moe._layout_name(self._wo) == "BlockScaledLayout"
        if decode and self._quantized:
            # a padding sequence (negative position) attends nothing
            attn = kv_attend(q, self.cache, cache_state, block_index=self.block_index, seq_block_ids=page_ids,
                             seq_lens=torch.where(positions < 0, 0, positions + sl), scale=float(scale),
                             softcap=self.softcap, out_dtype=torch.float16 if direct else h.dtype).view(bs, sl, H * hd)
        elif decode:
            # positions to attend: everything up to and including the new row (what the
            # reference's decode mask leaves unmasked)
            seq_lens = (positions + 1).contiguous()
            max_len = page_ids.shape[1] * stride
            out = torch.empty(bs, H * hd, dtype=torch.float16 if direct else h.dtype, device=dev)
            nbytes = C.lib.b200moe_attn_decode_scratch_bytes(ctypes.byref(self._desc), bs, H, max_len)
            # per call, as the layer's workspace: other streams and captured graphs have their own
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            with torch.cuda.device(dev):
                C.check(C.lib.b200moe_attn_decode(
                    _p(q), _DT[q.dtype], _p(slab), _DT[slab.dtype], ctypes.byref(self._desc), self.block_index,
                    _p(page_ids), _p(seq_lens), bs, page_ids.shape[1], H, max_len, float(scale),
                    float(self.softcap) if self.softcap is not None else 0.0, _p(out), _DT[out.dtype],
                    _p(scratch), nbytes, _moe._stream()), "attn_decode")
            attn = out.view(bs, 1, H * hd)
        else:
            kh = k.view(bs, sl, Hkv, hd)
            vh = v.view(bs, sl, Hkv, hd)
            before = int(start_index) if self._quantized else 0
            if before:  # a continued prompt: the cached positions, then the new ones as they are
                kc, vc = kv_read(self.cache, cache_state, block_index=self.block_index, seq_block_ids=page_ids,
                                 seq_lens=torch.full((bs,), before, device=dev, dtype=torch.int32), max_seq_len=before,
                                 dtype=q.dtype)
                kh, vh = torch.cat([kc, kh], dim=1), torch.cat([vc, vh], dim=1)
            if own:
                cu = torch.arange(bs + 1, device=dev, dtype=torch.int32)
                if attention_mask is not None:
                    _check_causal(attention_mask, bs, new_lens, dev)
                rows = lambda x, heads: x.reshape(-1, heads, hd)
                attn = prompt_attend(rows(q, H), rows(kh, Hkv), rows(vh, Hkv), cu_seqlens=cu * sl,
                                     cu_seqlens_k=cu * (before + sl) if before else None, scale=float(scale),
                                     softcap=self.softcap, out_dtype=torch.float16 if direct else q.dtype)
            else:
                attn = self._torch_attention(q.view(bs, sl, H, hd), kh, vh, attention_mask, before, scale)
            attn = attn.reshape(bs, sl, H * hd)
        if fused_out:
            y, = _moe.linear_rows(attn.reshape(bs * sl, H * hd), [_moe.prepare_linear(self._wo)],
                                  residual=hc.view(bs * sl, d), out_dtype=h.dtype)
            return y.view(bs, sl, d)
        y = self._linear(attn, self._wo, self._bias["attn_output"])
        if self._out_norm_w is not None:
            y = self._norm(y.contiguous(), self._out_norm_w)
        return h + y


def patch_attention_blocks(model, attention_kernel: Optional[str] = None) -> int:
    """Replaces every PagedLlamaAttentionBlock-shaped child of `model` (anything
    with `.theta`, `.cache`, `.head_count_kv` and `.block_index`) by a
    B200PagedAttentionBlock built from the same theta and cache, with the child's
    `attention_kernel` or the one given ("b200").  Returns the number of blocks
    replaced."""
    replaced = 0
    for parent in list(model.modules()):
        for name, child in list(parent.named_children()):
            if isinstance(child, B200PagedAttentionBlock):
                continue
            if not all(hasattr(child, a) for a in ("theta", "cache", "head_count_kv", "block_index", "attn_norm")):
                continue
            new = B200PagedAttentionBlock(
                child.theta, block_index=child.block_index, cache=child.cache, head_count=child.head_count,
                head_dim=child.head_dim, head_count_kv=child.head_count_kv, rms_epsilon=child.attn_norm.epsilon,
                attention_kernel=attention_kernel or getattr(child, "attention_kernel", "decomposed"),
                attention_scale=getattr(child, "attention_scale", None), softcap=getattr(child, "softcap", None))
            setattr(parent, name, new)
            replaced += 1
    return replaced
