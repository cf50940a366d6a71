"""A layer over 4-bit caches as it is used: prompts, a later chunk, decode steps (called and replayed by
DecodeGraphRunner) and a verification step, through Attention and attention_with_prologue, the
caches followed by the oracle."""
import numpy as np
import pytest
import torch

from fp4_utils import assert_close
from gpu_utils import say
from nanovllm_amd import (Attention, Fp4Cache, attention_with_prologue, flash_attn_with_kvcache,
                          paged_decode_with_prologue, qk_norm_rope_store, rope_cos_sin_cache,
                          store_kvcache)
from nanovllm_amd.engine.graph_runner import DecodeGraphRunner
from nanovllm_amd.utils.context import reset_context, set_context
from oracle import fp4_oracle as orc

pytestmark = pytest.mark.gpu

HQ, HKV, HD, BS, NB = 16, 8, 128, 256, 12
SCALE = HD ** -0.5
TABLES = [[7, 2], [11, 4], [0, 9]]


class _Norm:
    def __init__(self, weight):
        self.weight, self.eps = weight, 1e-6


class _Rope:
    cos_sin_cache = None


class _Model:
    """One layer with its caches on the GPU and in the oracle."""

    def __init__(self):
        gen = torch.Generator().manual_seed(5)
        w = (1 + 0.2 * torch.randn(2, HD, generator=gen)).to(torch.bfloat16).cuda()
        self.q_norm, self.k_norm, self.rope = _Norm(w[0]), _Norm(w[1]), _Rope()
        self.rope.cos_sin_cache = rope_cos_sin_cache(HD, 4096, 1e6, "cuda")
        self.attn = Attention(HQ, HD, SCALE, HKV)
        self.attn.k_cache, self.attn.v_cache = (Fp4Cache.zeros(NB, BS, HKV, HD) for _ in range(2))
        self.np = [(c.data.cpu().numpy(), c.scale.cpu().numpy())
                   for c in (self.attn.k_cache, self.attn.v_cache)]
        self.gen = gen

    def qkv(self, n):
        x = torch.randn(n, (HQ + 2 * HKV) * HD, generator=self.gen) * 2
        return x.to(torch.bfloat16).cuda()

    def rows(self, positions, qkv):
        """The layer's q, k, v after norms and rotation."""
        return qk_norm_rope_store(positions, qkv, HQ, HKV, HD, self.q_norm.weight,
                                  self.k_norm.weight, 1e-6, self.rope.cos_sin_cache)

    def store(self, k, v, slots):
        for i, x in enumerate((k, v)):
            orc.store(x.double().cpu().numpy(), *self.np[i], slots, i == 0)

    def check_caches(self):
        for c, (data, scale) in zip((self.attn.k_cache, self.attn.v_cache), self.np):
            np.testing.assert_array_equal(c.data.cpu().numpy(), data)
            np.testing.assert_array_equal(c.scale.cpu().numpy().view(np.uint16),
                                          scale.view(np.uint16))

    def attend(self, q, news, lens):
        """Oracle over what the caches hold."""
        qn, outs, sizes, at = q.double().cpu().numpy(), [], [], 0
        values = [orc.values(*self.np[i], keys=i == 0) for i in range(2)]
        pages = orc.through_pages(max(news), HQ // HKV, HD, len(news) * HKV, max(lens))
        for b, (n, m) in enumerate(zip(news, lens)):
            p = np.arange(m)
            rows = np.asarray(TABLES[b])[p // BS], p % BS
            o, s = orc.attention(qn[at:at + n], values[0][rows], values[1][rows], m, SCALE, pages)
            outs.append(o)
            sizes.append(s)
            at += n
        return np.concatenate(outs), np.concatenate(sizes)

    def layer(self, positions, qkv):
        return attention_with_prologue(self.attn, positions, qkv, self.q_norm, self.k_norm,
                                       self.rope)


def _slots(b, positions):
    return [TABLES[b][p // BS] * BS + p % BS for p in positions]


def _int(a, dtype=torch.int32):
    return torch.as_tensor(np.asarray(a)).to(dtype).cuda()


def _prefill_context(news, lens, with_tables):
    cu = lambda v: _int(np.concatenate([[0], np.cumsum(v)]))
    slots = [s for b, (n, m) in enumerate(zip(news, lens)) for s in _slots(b, range(m - n, m))]
    set_context(True, cu(news), cu(lens), max(news), max(lens), _int(slots), None,
                _int(TABLES) if with_tables else None)
    return slots, _int([p for n, m in zip(news, lens) for p in range(m - n, m)], torch.int64)


def test_a_layer_over_4_bit_caches():
    m = _Model()
    try:
        # prompts: stored in 4 bits, attended as they are
        lens = [70, 5, 330]
        slots, pos = _prefill_context(lens, lens, False)
        qkv = m.qkv(sum(lens))
        say("fp4 layer: prompts")
        out = m.layer(pos, qkv)
        q, k, v = m.rows(pos, qkv)
        plain = Attention(HQ, HD, SCALE, HKV)           # no cache: the same dense attention
        assert torch.equal(out, plain(q, k, v))
        m.store(k, v, slots)
        m.check_caches()

        # the next chunk of each, over what the caches hold; the module called by itself
        for news in ([100, 1, 20], [3, 8, 1]):
            lens = [a + b for a, b in zip(lens, news)]
            slots, pos = _prefill_context(news, lens, True)
            qkv = m.qkv(sum(news))
            q, k, v = m.rows(pos, qkv)
            say(f"fp4 layer: chunks {news}")
            out = m.attn(q, k, v)
            m.store(k, v, slots)
            m.check_caches()
            ref, size = m.attend(q, news, lens)
            assert_close(out, ref, size, "bf16", f"fp4 layer, chunks {news}")

        # decode steps
        for step in range(2):
            lens = [n + 1 for n in lens]
            slots = [_slots(b, [n - 1])[0] for b, n in enumerate(lens)]
            set_context(False, slot_mapping=_int(slots), context_lens=_int(lens),
                        block_tables=_int(TABLES))
            pos, qkv = _int([n - 1 for n in lens], torch.int64), m.qkv(3)
            say(f"fp4 layer: decode {step}")
            out = m.layer(pos, qkv)
            q, k, v = m.rows(pos, qkv)
            m.store(k, v, slots)
            m.check_caches()
            ref, size = m.attend(q, [1] * 3, lens)
            assert out.shape == (3, 1, HQ, HD)
            assert_close(out, ref, size, "bf16", f"fp4 layer, decode {step}")
    finally:
        reset_context()

    # verification: 4 drafts and the last accepted token
    n = 5
    lens = [x + n - 1 for x in lens]
    q = m.qkv(3 * n)[:, :HQ * HD].view(3, n, HQ, HD)
    k, v = (m.qkv(3 * (n - 1))[:, :HKV * HD].reshape(-1, HKV, HD) for _ in range(2))
    slots = [s for b, x in enumerate(lens) for s in _slots(b, range(x - n + 1, x))]
    store_kvcache(k, v, m.attn.k_cache, m.attn.v_cache, _int(slots))
    out = flash_attn_with_kvcache(q, m.attn.k_cache, m.attn.v_cache, cache_seqlens=_int(lens),
                                  block_table=_int(TABLES), softmax_scale=SCALE, causal=True)
    m.store(k, v, slots)
    m.check_caches()
    ref, size = m.attend(q.flatten(0, 1), [n] * 3, lens)
    assert_close(out, ref, size, "bf16", "fp4 layer, verification")


def test_decode_steps_replayed_as_a_graph():
    """DecodeGraphRunner with buckets of 1 to 4 over live batches of 3, 1 and 2 sequences."""
    m = _Model()
    prompts = [300, 256, 20]
    try:
        slots, pos = _prefill_context(prompts, prompts, False)
        qkv = m.qkv(sum(prompts))
        m.layer(pos, qkv)
        _, k, v = m.rows(pos, qkv)
        m.store(k, v, slots)
        reset_context()
        step = lambda positions, qkv: m.layer(positions, qkv).reshape(positions.numel(), HQ * HD)
        first = [(c.data[0].clone(), c.scale[0].clone()) for c in (m.attn.k_cache, m.attn.v_cache)]
        say("fp4 graph: capture")
        runner = DecodeGraphRunner(step, 4, 2, {"qkv": (((HQ + 2 * HKV) * HD,), torch.bfloat16)},
                                   ((HQ * HD,), torch.bfloat16))
        # capturing runs the step on zeroed metadata, which stores at slot 0
        for c, (data, scale) in zip((m.attn.k_cache, m.attn.v_cache), first):
            c.data[0].copy_(data)
            c.scale[0].copy_(scale)
        lens = list(prompts)
        for live in (3, 1, 2, 3):
            lens = [n + (b < live) for b, n in enumerate(lens)]
            now = lens[:live]
            slots = [_slots(b, [n - 1])[0] for b, n in enumerate(now)]
            set_context(False, slot_mapping=_int(slots), context_lens=_int(now),
                        block_tables=_int(TABLES[:live]))
            pos, qkv = _int([n - 1 for n in now], torch.int64), m.qkv(live)
            say(f"fp4 graph: replay {live}")
            out = runner.run(pos, qkv=qkv).clone()
            q, k, v = m.rows(pos, qkv)
            m.store(k, v, slots)
            m.check_caches()
            ref, size = m.attend(q, [1] * live, now)
            assert_close(out.view(live, HQ, HD), ref, size, "bf16", f"fp4 graph, {live} live")
    finally:
        reset_context()


def test_the_prologue_s_own_calls_take_the_caches():
    """qk_norm_rope_store and paged_decode_with_prologue into 4-bit caches are the calls that they
    stand for."""
    m = _Model()
    lens = [5, 300, 512]
    qkv = m.qkv(3)
    pos = torch.tensor([n - 1 for n in lens], device="cuda")
    slots = torch.tensor([TABLES[b][(n - 1) // BS] * BS + (n - 1) % BS for b, n in enumerate(lens)],
                         dtype=torch.int32, device="cuda")
    args = (pos, qkv, HQ, HKV, HD, m.q_norm.weight, m.k_norm.weight, 1e-6, m.rope.cos_sin_cache)
    caches = [[Fp4Cache.zeros(NB, BS, HKV, HD) for _ in range(2)] for _ in range(3)]
    q, k, v = qk_norm_rope_store(*args)
    store_kvcache(k, v, *caches[0], slots)
    got = qk_norm_rope_store(*args, *caches[1], slots)
    assert all(torch.equal(a, b) for a, b in zip(got, (q, k, v)))
    assert qk_norm_rope_store(*args, *caches[1], slots, return_k=False)[1] is None
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    tables = torch.tensor(TABLES, dtype=torch.int32, device="cuda")
    want = flash_attn_with_kvcache(q.unsqueeze(1), *caches[0], cache_seqlens=lens,
                                   block_table=tables, softmax_scale=SCALE, causal=True)
    out = torch.empty(3, HQ, HD, dtype=torch.bfloat16, device="cuda")
    paged_decode_with_prologue(*args, *caches[2], slots, lens, tables, SCALE, out=out)
    assert torch.equal(out, want[:, 0])
    for pair in caches[1:]:
        for c, ref in zip(pair, caches[0]):
            assert torch.equal(c.data, ref.data) and torch.equal(c.scale, ref.scale)
    say("prologue calls over 4-bit caches ok")
