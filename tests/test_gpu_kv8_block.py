"""B200PagedAttentionBlock with an 8-bit cache, query / key norms, the HuggingFace rotation
order and padding: prompts, continued prompts, steps of one and of several tokens, against
the formulas in 64 bits over the values that the cache holds."""
import pytest
import torch

from oracle import kv8_oracle as ko
from shark_platform_b200 import synthetic as syn

pytestmark = pytest.mark.gpu

I8, E4 = torch.int8, torch.float8_e4m3fn


class Model:
    def __init__(self, dtype, norms=False, use_hf=False, softcap=None, heads=4, kv_heads=2, act=torch.float32):
        if not torch.cuda.is_available():
            pytest.fail("GPU tests need a CUDA device")
        from shark_platform_b200 import attention as A, types as T

        self.A, self.hd, self.heads, self.kvh, self.softcap, self.use_hf, self.act = A, 64, heads, kv_heads, softcap, use_hf, act
        self.c = c = syn.make_attn_case(seed=31, hidden=heads * 64, head_count=heads, head_count_kv=kv_heads)
        gen = torch.Generator().manual_seed(32)
        P = lambda t: T.DefaultPrimitiveTensor(data=t.cuda())
        tree = {n: {"weight": P(t)} for n, t in (("attn_norm", c.norm_w), ("attn_q", c.wq), ("attn_k", c.wk),
                                                 ("attn_v", c.wv), ("attn_output", c.wo))}
        self.qn = self.kn = None
        if norms:
            self.qn, self.kn = (1 + 0.2 * torch.randn(64, generator=gen) for _ in range(2))
            tree["attn_q_norm"], tree["attn_k_norm"] = {"weight": P(self.qn)}, {"weight": P(self.kn)}
        self.cache = A.PagedKVCache(transformer_block_count=2, attn_head_count=kv_heads, attn_head_dim=64,
                                    block_seq_stride=16, dtype=dtype, device="cuda")
        self.block = A.B200PagedAttentionBlock(T.Theta(tree), block_index=1, cache=self.cache, head_count=heads, head_dim=64,
                                               head_count_kv=kv_heads, rms_epsilon=c.eps, softcap=softcap)
        self.rope = A.RotaryEmbeddingLayer(rope_dimension_count=64, max_seqlen=4096, use_hf=use_hf)
        self.freqs = 1.0 / (10000.0 ** (torch.arange(0, 64, 2).float() / 64))
        self.state = self.cache.allocate(12)
        self.ids = torch.randperm(12, generator=gen)[:10].view(2, 5)
        self.gen = gen

    def rows(self, sl):
        return torch.randn(2, sl, self.heads * 64, generator=self.gen).to(self.act)

    def call(self, h, **kw):
        return self.block(h.cuda().to(self.act), embedding=self.rope, cache_state=self.state, seq_block_ids=self.ids.cuda(), **kw)

    def held(self, b, n):
        """K and V of the first n positions of sequence b as the cache holds them."""
        if self.cache.quantized:
            codes, scales = ko.page_views(self.state, self.cache)
            return ko.gather(codes, scales, self.cache, 1, self.ids[b], n)
        slab = self.state[0].cpu().double().unflatten(1, self.cache.sub_page_dims)
        return torch.stack([slab[self.ids[b, p // 16], 1, :, p % 16] for p in range(n)], dim=1)

    def want(self, h, starts, fresh_from=None):
        """The block's output in 64 bits.  K and V: the cache's before position fresh_from[b]
        (None: all of it), the new rows themselves behind it.  Also the new rows."""
        c, out, new = self.c, [], []
        for b in range(2):
            x = h[b].double()
            n = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + c.eps) * c.norm_w.double()
            q, k, v = ((n @ w.double().T).unflatten(-1, (-1, 64)) for w in (c.wq, c.wk, c.wv))
            pos = starts[b] + torch.arange(len(h[b]))
            q = ko.turn(q, pos, self.freqs, self.qn, eps=c.eps, halves=self.use_hf)
            k = ko.turn(k, pos, self.freqs, self.kn, eps=c.eps, halves=self.use_hf)
            total = starts[b] + len(h[b])
            kk, vv = self.held(b, total)
            if fresh_from is not None:
                at = fresh_from[b]
                kk, vv = torch.cat([kk[:at], k]), torch.cat([vv[:at], v])
            o = ko.attend(q, kk, vv, [int(p) + 1 for p in pos], 64 ** -0.5, self.softcap)
            out.append(x + o.flatten(1) @ c.wo.double().T)
            new.append((k, v))
        return torch.stack(out), new


# fp32: as the block's other tests.  bf16: h, the normed rows, the weights, q / k / v, the rotated
# rows, the attention's rows, the projection's and the sum are rounded, half a step of 2^-8 at
# most and 2^-8 / sqrt(3) in the mean square each.  Eight of them in a row with independent
# errors are sqrt(8) 2^-8 / sqrt(3) = 6.4e-3 of the attention's part in the 2-norm, and the
# scores' own (of size 2, four roundings: 2 * 2 * 2^-8 / sqrt(3) = 9e-3 of each probability,
# averaged over more than one position) less than half of that again: within 1e-2.
TOL = {torch.float32: 2e-4, torch.bfloat16: 6e-2}
REL = 1e-2


def _near(got, want, act):
    off = got.cpu().double() - want
    if act == torch.float32:
        assert off.abs().max() < TOL[act], float(off.abs().max())
    else:
        assert off.norm() < REL * want.norm(), float(off.norm() / want.norm())


@pytest.mark.parametrize("act", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype,norms,use_hf,softcap,heads,kv_heads", [
    (I8, False, False, None, 4, 2), (E4, True, True, None, 4, 2), (I8, True, False, 30.0, 4, 1), (E4, False, True, 30.0, 12, 1)])
def test_eight_bit_block(act, dtype, norms, use_hf, softcap, heads, kv_heads):
    from shark_platform_b200 import moe

    m = Model(dtype, norms, use_hf, softcap, heads, kv_heads, act)
    h = m.rows(20)
    y = m.call(h, start_index=0)
    want, new = m.want(h, [0, 0], [0, 0])
    _near(y, want, act)
    for b in range(2):  # the cache holds what was computed, to its precision
        for got, x in zip(m.held(b, 20), new[b]):
            step = x.abs().amax() * (1 / 127 if dtype == I8 else 2.0 ** -4)
            assert (got - x).abs().max() <= step * 0.6 + TOL[act]
    # the prompt goes on: the cached positions are attended
    h = m.rows(13)
    _near(m.call(h, start_index=20), m.want(h, [20, 20], [20, 20])[0], act)
    mask = torch.zeros(2, 1, 7, 7).masked_fill_(torch.ones(7, 7, dtype=torch.bool).triu(1), float("-inf")).cuda()
    h = m.rows(7)
    _near(m.call(h, start_index=33, attention_mask=mask), m.want(h, [33, 33], [33, 33])[0], act)
    # steps: ragged positions, several tokens at once
    at = [40, 36]
    for sl in (1, 1, 4, 16):
        h = m.rows(sl)
        y = m.call(h, start_positions=torch.tensor(at).cuda())
        _near(y, m.want(h, at)[0], act)
        at = [p + sl for p in at]
    # a padding sequence beside a live one
    h = m.rows(1)
    before = [t.clone() for t in m.state]
    y = m.call(h, start_positions=torch.tensor([at[0], -1]).cuda())
    want, _ = m.want(h, [at[0], 0])
    _near(y[0], want[0], act)
    assert torch.isfinite(y[1]).all()
    pages = m.ids[1].cuda()
    assert all(torch.equal(a[pages].view(torch.uint8), b[pages].view(torch.uint8)) for a, b in zip(m.state, before))
    assert moe.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("norms,use_hf", [(True, False), (False, True), (True, True)])
def test_norms_and_order_with_a_plain_cache(dtype, norms, use_hf):
    from shark_platform_b200 import moe

    act = torch.float32 if dtype == torch.float32 else torch.bfloat16
    m = Model(dtype, norms, use_hf, act=act)
    h = m.rows(32)
    _near(m.call(h, start_index=0), m.want(h, [0, 0], [0, 0])[0], act)
    at = [32, 20]
    for _ in range(2):
        h = m.rows(1)
        _near(m.call(h, start_positions=torch.tensor(at).cuda()), m.want(h, at)[0], act)
        at = [p + 1 for p in at]
    assert moe.device_status() == 0


@pytest.mark.parametrize("dtype", [I8, torch.float32])
def test_padding_of_a_prompt_stays_out_of_the_cache(dtype):
    m = Model(dtype)
    h = m.rows(32)
    lens = torch.tensor([32, 19])
    m.call(h, start_index=0, new_lens=lens.cuda())
    live = m.held(1, 19)
    h2 = h.clone()
    h2[1, 19:] = 1e4
    state = [t.clone() for t in m.state]
    for t in m.state:
        t.zero_()
    m.call(h2, start_index=0, new_lens=lens.cuda())
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(m.state, state))
    assert (live != 0).any()


def test_refusals():
    from shark_platform_b200 import _cabi as C, types as T

    m = Model(I8)
    with pytest.raises(C.B200MoeError, match="at most 16"):
        m.call(m.rows(17), start_positions=torch.tensor([0, 0]).cuda())
    with pytest.raises(C.B200MoeError, match="new_lens"):
        m.call(m.rows(1), start_positions=torch.tensor([0, 0]).cuda(), new_lens=torch.tensor([1, 0]).cuda())
    with pytest.raises(C.B200MoeError, match="8-bit codes"):
        m.block(m.rows(1).cuda(), embedding=m.rope, cache_state=m.state[:1], seq_block_ids=m.ids.cuda(), start_index=0)
    plain = Model(torch.float32)
    with pytest.raises(C.B200MoeError, match="one token"):
        plain.call(plain.rows(2), start_positions=torch.tensor([0, 0]).cuda())
