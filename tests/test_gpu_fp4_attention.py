"""Attention over the 4-bit cache on the GPU against the oracle in 64 bits, within bounds that follow
from the types (oracle.fp4_oracle.attention)."""
import numpy as np
import pytest
import torch

from fp4_utils import DTYPES, Pages, assert_close, rng_rows, tables_of
from gpu_utils import say
from nanovllm_amd import (Fp4Cache, flash_attn_varlen_func, flash_attn_with_kvcache, load_kvcache,
                          paged_decode, store_kvcache, varlen_prefill)
from oracle import fp4_oracle as orc

pytestmark = pytest.mark.gpu


def _reference(q, pages, tables, n_queries, lens, scale, keys=None):
    """Oracle of sequences whose queries follow each other in q [tokens, Hq, D]; keys: the most that
    the call was told of, what the table holds if none."""
    qn = q.double().cpu().numpy()
    keys = keys or len(tables[0]) * pages.bs
    through = orc.through_pages(max(n_queries), q.shape[1] // pages.hkv, pages.d,
                                len(lens) * pages.hkv, keys)
    out, size = np.zeros(qn.shape), np.zeros(qn.shape)
    at = 0
    for b, (n, m) in enumerate(zip(n_queries, lens)):
        k, v = pages.rows(tables[b], m)
        out[at:at + n], size[at:at + n] = orc.attention(qn[at:at + n], k, v, m, scale, through)
        at += n
    return out, size


def _wide(tables, bs, tokens):
    """The tables with room for `tokens`: chunks enough for the route over f16 pages."""
    wide = np.full((len(tables), -(-tokens // bs)), -1, np.int32)
    wide[:, :tables.shape[1]] = tables
    return wide


def _random_pages(seed, nb, bs, hkv, d):
    """Caches of random codes and scales (nothing to quantise)."""
    rng = np.random.default_rng(seed)
    pages = Pages.__new__(Pages)
    pages.nb, pages.bs, pages.hkv, pages.d = nb, bs, hkv, d
    pages.np = [(rng.integers(0, 256, (nb, hkv, bs, d // 2), dtype=np.uint8),
                 rng.uniform(0.1, 0.4, (nb, hkv, d // 32, bs)).astype(np.float16)) for _ in range(2)]
    return pages


def _int(a):
    return torch.as_tensor(np.asarray(a, dtype=np.int32)).cuda()


LADDER = [1, 0, 15, 16, 17, 63, 64, 65, 255, 256, 257, 1000]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv,d,bs", [(16, 8, 128, 256), (16, 16, 128, 64), (16, 4, 128, 256),
                                         (16, 2, 128, 256), (12, 4, 128, 48), (16, 1, 128, 16),
                                         (8, 4, 64, 256), (8, 1, 64, 16), (3, 1, 64, 32)])
def test_decode_over_a_ladder_of_contexts(hq, hkv, d, bs, dtype):
    tables, nb = tables_of(LADDER, bs, 1)
    pages = Pages(5, nb, bs, hkv, d, dtype)
    q = rng_rows(9, (len(LADDER), hq, d), dtype).cuda()
    say(f"fp4 decode ladder {hq}/{hkv} x {d} pages {bs} {dtype}")
    out = paged_decode(q, *pages.gpu(), _int(LADDER), _int(tables), d ** -0.5)
    ref, size = _reference(q, pages, tables, [1] * len(LADDER), LADDER, d ** -0.5)
    assert not out[1].any()                        # no key: zeros
    assert_close(out, ref, size, dtype, "fp4 decode ladder")


@pytest.mark.parametrize("lens", [[5000], [1500, 3000], [64], [2100] * 3 + [1] * 30])
@pytest.mark.parametrize("bs", [256, 16])
def test_decode_of_contexts_cut_into_many_parts(lens, bs):
    tables, nb = tables_of(lens, bs, 2)
    pages = Pages(6, nb, bs, 2, 128)
    q = rng_rows(3, (len(lens), 4, 128), "bf16").cuda()
    say(f"fp4 decode {lens[:4]} pages {bs}")
    out = paged_decode(q, *pages.gpu(), _int(lens), _int(tables), None)
    ref, size = _reference(q, pages, tables, [1] * len(lens), lens, 128 ** -0.5)
    assert_close(out, ref, size, "bf16", "fp4 decode parts")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,hq,hkv,d", [(2, 16, 8, 128), (6, 16, 8, 128), (8, 16, 8, 128),
                                        (5, 8, 1, 128), (33, 4, 2, 128), (70, 4, 2, 128), (3, 4, 4, 64),
                                        (70, 2, 2, 64)])
def test_several_queries_of_every_sequence(n, hq, hkv, d, dtype):
    lens = [n, n + 1, 64, 300, 130, max(0, n - 1), 0]     # two with rows that see no key
    tables, nb = tables_of(lens, 64, 4)
    pages = Pages(7, nb, 64, hkv, d, dtype)
    q = rng_rows(11, (len(lens), n, hq, d), dtype).cuda()
    say(f"fp4 {n} queries {hq}/{hkv} x {d} {dtype}")
    ref, size = _reference(q.flatten(0, 1), pages, tables, [n] * len(lens), lens, d ** -0.5)
    # a workgroup per group, and (tables that could hold more) ranges of chunks
    for table in (tables, _wide(tables, 64, 5000)):
        out = flash_attn_with_kvcache(q, *pages.gpu(), cache_seqlens=_int(lens),
                                      block_table=_int(table), causal=True)
        assert out.shape == q.shape
        assert_close(out, ref, size, dtype, "fp4 several queries")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("bs", [256, 16])
@pytest.mark.parametrize("news,cached", [([3, 0, 40, 1, 9], [0, 70, 5, 300, 64]),
                                         ([200, 17], [100, 0]), ([1], [1])])
def test_ragged_queries(news, cached, bs, dtype):
    hq, hkv, d = 8, 4, 128
    lens = [a + b for a, b in zip(news, cached)]
    tables, nb = tables_of(lens, bs, 8)
    pages = Pages(12, nb, bs, hkv, d, dtype)
    total = sum(news)
    # two rows behind the last sequence stay as they were
    out = torch.full((total + 2, hq, d), 7.0, dtype=DTYPES[dtype], device="cuda")
    q = rng_rows(13, (total + 2, hq, d), dtype).cuda()
    cu = lambda v: _int(np.concatenate([[0], np.cumsum(v)]))
    say(f"fp4 ragged {news} pages {bs} {dtype}")
    varlen_prefill(q, *pages.gpu(), cu(news), cu(lens), max(news), None, block_table=_int(tables),
                   out=out)
    ref, size = _reference(q[:total], pages, tables, news, lens, d ** -0.5)
    assert_close(out[:total], ref, size, dtype, "fp4 ragged")
    assert (out[total:] == 7.0).all()
    got = flash_attn_varlen_func(q, *pages.gpu(), cu(news), cu(lens), max(news), max(lens),
                                 causal=True, block_table=_int(tables))
    assert torch.equal(got[:total], out[:total])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,hq,hkv,d,bs", [(9, 16, 8, 128, 64), (16, 16, 8, 128, 16),
                                           (60, 16, 8, 128, 256), (30, 8, 8, 64, 64),
                                           (4, 64, 8, 64, 16), (25, 8, 8, 128, 48),
                                           (50, 16, 8, 128, 64)])
def test_tiles_of_32_rows(n, hq, hkv, d, bs, dtype):
    """Tables that could hold 32768 tokens of each sequence: many chunks for every wave, by which tiles
    of 32 rows are chosen, over contexts that end anywhere."""
    lens = [n, n + 1, 64, 300, 130, n - 1, 0, 1000]
    tables, nb = tables_of(lens, bs, 4)
    wide = np.full((len(lens), 32768 // bs), -1, np.int32)
    wide[:, :tables.shape[1]] = tables
    pages = Pages(7, nb, bs, hkv, d, dtype)
    q = rng_rows(11, (len(lens), n, hq, d), dtype).cuda()
    say(f"fp4 tiles of 32 rows: {n} queries {hq}/{hkv} x {d} pages {bs} {dtype}")
    out = flash_attn_with_kvcache(q, *pages.gpu(), cache_seqlens=_int(lens), block_table=_int(wide),
                                  causal=True)
    ref, size = _reference(q.flatten(0, 1), pages, tables, [n] * len(lens), lens, d ** -0.5)
    assert_close(out, ref, size, dtype, "fp4 tiles of 32 rows")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("n,hq,hkv,d,bs,width", [(1, 16, 8, 128, 256, 0), (3, 16, 8, 128, 16, 0),
                                                 (6, 16, 8, 128, 64, 0), (1, 16, 2, 128, 256, 0),
                                                 (12, 16, 8, 128, 256, 65536), (2, 8, 8, 64, 32, 0),
                                                 (20, 8, 8, 64, 64, 65536)])
def test_several_chunks_for_every_wave(n, hq, hkv, d, bs, width, dtype):
    """More chunks of 64 keys than the 2048 waves: groups that waves of a workgroup share, that
    workgroups share, and whole ones.  (Caches of random codes; width: tokens that a table could hold.)"""
    mean = 64 * 2900 // (6 * hkv)
    lens = [int(mean * x) for x in (0.02, 1.9, 0.3, 1, 1.5, 0.7)] + [0, n]
    tables, nb = tables_of(lens, bs, 4)
    pages = _random_pages(8, nb, bs, hkv, d)
    wide = np.full((len(lens), max(width // bs, tables.shape[1])), -1, np.int32)
    wide[:, :tables.shape[1]] = tables
    q = rng_rows(11, (len(lens), n, hq, d), dtype).cuda()
    say(f"fp4 {n} queries {hq}/{hkv} x {d} pages {bs} {dtype}, several chunks a wave")
    out = flash_attn_with_kvcache(q, *pages.gpu(), cache_seqlens=_int(lens), block_table=_int(wide),
                                  causal=True)
    ref, size = _reference(q.flatten(0, 1), pages, tables, [n] * len(lens), lens, d ** -0.5)
    assert_close(out, ref, size, dtype, "fp4 several chunks a wave")


@pytest.mark.parametrize("batch,n,hq,hkv,d,most,ragged", [
    (70, 1, 16, 8, 128, 1000, True), (40, 1, 16, 8, 128, 1500, True), (33, 3, 16, 8, 128, 700, True),
    (64, 6, 16, 8, 128, 600, True), (128, 1, 3, 3, 128, 800, False), (128, 1, 6, 3, 64, 1300, True),
    (129, 1, 4, 2, 128, 700, False), (2, 1, 256, 256, 64, 600, True), (3, 1, 130, 130, 64, 600, True)])
def test_more_groups_than_cus_of_short_contexts(batch, n, hq, hkv, d, most, ragged):
    """Sequences are dealt out by their length: every one of them once, whatever lengths are alike,
    zero, or given with prefix sums that leave some without queries."""
    rng = np.random.default_rng(batch)
    lens = [int(x) for x in rng.integers(0, most // 64 // 3, batch) * 64 + rng.integers(0, 2, batch) * 3]
    lens[1], lens[-1] = most, 0
    news = [n if not ragged or i % 5 else 0 for i in range(batch)]
    tables, nb = tables_of(lens, 64, 4)
    pages = _random_pages(8, nb, 64, hkv, d)
    q = rng_rows(11, (sum(news), hq, d), "bf16").cuda()
    say(f"fp4 {batch} x {n} queries {hq}/{hkv} x {d}, dealt out by length")
    if ragged:
        cu = lambda v: _int(np.concatenate([[0], np.cumsum(v)]))
        out = flash_attn_varlen_func(q, *pages.gpu(), cu(news), cu(lens), n, most, causal=True,
                                     block_table=_int(tables))
    else:
        out = paged_decode(q, *pages.gpu(), _int(lens), _int(tables), None)
    ref, size = _reference(q, pages, tables, news, lens, d ** -0.5)
    assert_close(out, ref, size, "bf16", "fp4 dealt out by length")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv,d,bs", [(16, 8, 128, 256), (4, 1, 128, 16), (16, 16, 64, 48)])
def test_one_workgroup_per_group_and_ranges_of_waves_agree(hq, hkv, d, bs, dtype):
    """Short contexts in one kernel; the same with a table that could hold more, cut between waves."""
    lens = [1, 0, 64, 700, 1000, 65]
    tables, nb = tables_of(lens, bs, 4)
    pages = Pages(7, nb, bs, hkv, d, dtype)
    q = rng_rows(11, (len(lens), hq, d), dtype).cuda()
    ref, size = _reference(q, pages, tables, [1] * len(lens), lens, d ** -0.5)
    for width in (tables.shape[1], 8192 // bs):
        wide = np.full((len(lens), width), -1, np.int32)
        wide[:, :tables.shape[1]] = tables
        out = paged_decode(q, *pages.gpu(), _int(lens), _int(wide), None)
        assert_close(out, ref, size, dtype, f"fp4 decode, tables of {width} pages")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hq,hkv,bs", [(2, 2, 256), (4, 2, 16), (4, 1, 64), (8, 1, 48), (3, 1, 64)])
def test_chunks_of_many_queries(hq, hkv, bs, dtype):
    """Over f16 pages (three heads per kv head: without), with chunks that end inside a tile, in front
    of everything, and sequences without queries or with fewer keys than queries."""
    news, cached = [200, 33, 0, 64, 40], [300, 0, 20, 65, -10]
    lens = [a + b for a, b in zip(news, cached)]
    tables, nb = tables_of(lens, bs, 8)
    tables = _wide(tables, bs, 32768)
    pages = Pages(12, nb, bs, hkv, 128, dtype)
    q = rng_rows(13, (sum(news), hq, 128), dtype).cuda()
    cu = lambda v: _int(np.concatenate([[0], np.cumsum(v)]))
    say(f"fp4 chunks {hq}/{hkv} pages {bs} {dtype}")
    for mk in (None, 20000, max(lens)):             # the last: without pages
        out = varlen_prefill(q, *pages.gpu(), cu(news), cu(lens), max(news), None,
                             block_table=_int(tables), max_seqlen_k=mk)
        ref, size = _reference(q, pages, tables, news, lens, 128 ** -0.5, mk)
        assert_close(out, ref, size, dtype, "fp4 chunks")


@pytest.mark.parametrize("up", [2.0 ** 20, 2.0 ** -20])
def test_chunks_of_queries_far_from_one(up):
    """bf16 queries outside f16's range, and values that only an eighth of fits it."""
    hq, hkv, n = 2, 1, 100
    tables, nb = tables_of([120], 64, 8)
    tables = _wide(tables, 64, 98304)
    pages = Pages(12, nb, 64, hkv, 128)
    big = rng_rows(3, (nb * 64, hkv, 128), "bf16").double().numpy() * 2.0 ** 16
    orc.store(big, *pages.np[1], np.arange(nb * 64), False)
    q = (rng_rows(13, (n, hq, 128), "bf16") * up).cuda()
    scale = 128 ** -0.5 / up
    out = flash_attn_with_kvcache(q[None], *pages.gpu(), cache_seqlens=_int([120]),
                                  block_table=_int(tables), softmax_scale=scale, causal=True)
    ref, size = _reference(q, pages, tables, [n], [120], scale)
    assert_close(out[0], ref, size, "bf16", "fp4 far queries")


def test_chunks_do_not_see_what_is_not_finite_behind_the_mask():
    n, lens = 100, [130]
    tables, nb = tables_of(lens, 64, 4)
    tables = _wide(tables, 64, 65536)
    pages = Pages(7, nb, 64, 2, 128)
    q = rng_rows(1, (n, 4, 128), "bf16").cuda()
    ref, size = _reference(q, pages, tables, [n], lens, 128 ** -0.5)
    for i in range(2):                                # key 90: head 0's key, head 1's value
        pages.np[i][1][tables[0][1], i, 2, 90 - 64] = np.nan
    out = flash_attn_with_kvcache(q[None], *pages.gpu(), cache_seqlens=_int(lens),
                                  block_table=_int(tables), causal=True)[0]
    sees = 90 - (130 - n)                             # the first query that sees it
    assert torch.isnan(out[sees:]).all()
    assert_close(out[:sees], ref[:sees], size[:sees], "bf16", "fp4 chunk, masked NaN")


def test_a_batch_larger_than_the_pages_goes_in_parts():
    """Tables of 16384 tokens: 64 MiB of f16 keys and values for a sequence, so 8 at a time."""
    lens, n = [40, 300, 17, 90, 33, 50, 64, 65, 129, 200, 35], 100
    tables, nb = tables_of(lens, 256, 4)
    pages = Pages(7, nb, 256, 8, 128)
    wide = np.full((len(lens), 64), -1, np.int32)
    wide[:, :tables.shape[1]] = tables
    q = rng_rows(1, (len(lens), n, 16, 128), "bf16").cuda()
    say("fp4 chunks in parts")
    out = flash_attn_with_kvcache(q, *pages.gpu(), cache_seqlens=_int(lens), block_table=_int(wide),
                                  causal=True)
    ref, size = _reference(q.flatten(0, 1), pages, wide, [n] * len(lens), lens, 128 ** -0.5)
    assert_close(out, ref, size, "bf16", "fp4 parts of a batch")


def test_a_chunk_over_more_keys_than_one_grid_dimension_holds():
    """More than 32768 pieces of 16 keys.  Query i's key, 30 / |q| times the query, is the only one with
    weight: scores of 25 and more against N(0, 1), so the others weigh 525288 e^(0.5 - 25), 1e-5."""
    n, keys, d, bs = 200, 16 * 32768 + 1000, 128, 256
    gen = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
    q = rand(n, 1, d).to(torch.bfloat16)
    at = torch.arange(n, device="cuda") * 4 + keys - 1000 - 100     # both sides of key 524288
    k, v = (rand(keys, 1, d).to(torch.bfloat16) for _ in range(2))
    k[at] = (30 * q / q.float().norm(dim=-1, keepdim=True)).to(torch.bfloat16)
    caches = [Fp4Cache.zeros(-(-keys // bs), bs, 1, d) for _ in range(2)]
    slots = torch.arange(keys, dtype=torch.int32, device="cuda")
    store_kvcache(k, v, *caches, slots)
    say("fp4 chunk over 525288 keys")
    out = flash_attn_with_kvcache(q[None], *caches, cache_seqlens=_int([keys]), causal=True,
                                  block_table=_int(np.arange(-(-keys // bs))[None]))[0]
    want = load_kvcache(*caches, slots[at], torch.float16)[1].float()
    # the output's rounding, three of f16 (page, probability, the values compared with), the others
    bound = (2.0 ** -8 + 3 * 2.0 ** -11) * want.abs() + 1e-4
    assert ((out.float() - want).abs() <= bound).all()


def test_a_captured_chunk_follows_its_inputs():
    lens, n = [130, 190], 100
    tables, nb = tables_of([190] * 2, 64, 3)
    tables = _wide(tables, 64, 32768)
    pages = Pages(7, nb, 64, 2, 128)
    q, keys = rng_rows(1, (2, n, 4, 128), "bf16").cuda(), _int(lens)
    call = lambda: flash_attn_with_kvcache(q, *gpu, cache_seqlens=keys, block_table=bt, causal=True)
    gpu, bt = pages.gpu(), _int(tables)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i, now in enumerate([lens, [90, 101], [190, 190], lens]):
        q.copy_(rng_rows(20 + i, (2, n, 4, 128), "bf16"))
        keys.copy_(_int(now))
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        ref, size = _reference(q.flatten(0, 1), pages, tables, [n] * 2, now, 128 ** -0.5)
        assert_close(out, ref, size, "bf16", f"fp4 chunk replay {i}")


def test_queries_and_outputs_with_strides():
    lens = [77, 130]
    tables, nb = tables_of(lens, 64, 4)
    pages = Pages(7, nb, 64, 2, 128)
    wide = rng_rows(1, (2, 3, 4 * 128 + 64), "bf16").cuda()
    q = wide[:, 1, 32:32 + 512].view(2, 4, 128)
    buf = torch.full((2, 4, 160), 3.0, dtype=torch.bfloat16, device="cuda")
    table = torch.full((2, 7), -1, dtype=torch.int64, device="cuda")
    table[:, 1:1 + tables.shape[1]] = _int(tables)
    paged_decode(q, *pages.gpu(), _int(lens).long(), table[:, 1:], 0.1, out=buf[:, :, 16:144])
    ref, size = _reference(q, pages, tables, [1, 1], lens, 0.1)
    assert_close(buf[:, :, 16:144], ref, size, "bf16", "fp4 strides")
    assert (buf[:, :, :16] == 3.0).all() and (buf[:, :, 144:] == 3.0).all()


def test_what_lies_past_a_context_or_behind_the_mask_does_not_count():
    """NaN and infinite scales in a page's slots past the context, and NaN in a key that only the
    later query sees."""
    lens, n = [40, 100], 2
    tables, nb = tables_of(lens, 64, 4)
    pages = Pages(7, nb, 64, 2, 128)
    q = rng_rows(1, (2, n, 4, 128), "bf16").cuda()
    ref, size = _reference(q.flatten(0, 1), pages, tables, [n, n], lens, 128 ** -0.5)
    for i in range(2):
        for b, m in enumerate(lens):
            page, off = tables[b][(m - 1) // 64], (m - 1) % 64
            pages.np[i][1][page, :, :, off + 1:] = np.nan if b else np.inf
            pages.np[i][0][page, :, off + 1:] = 0xFF
            pages.np[i][1][page, 0, :, off] = np.nan     # the last key of head 0
    out = flash_attn_with_kvcache(q, *pages.gpu(), cache_seqlens=_int(lens),
                                  block_table=_int(tables), causal=True).cpu()
    assert torch.isnan(out[:, 1, :2]).all()          # the query that sees it, heads of kv head 0
    keep = np.ones((2, n, 4), bool)
    keep[:, 1, :2] = False
    ref, size = ref.reshape(2, n, 4, 128), size.reshape(2, n, 4, 128)
    assert_close(out[torch.from_numpy(keep)], ref[keep], size[keep], "bf16", "fp4 masked NaN")


def test_a_value_that_is_not_finite_stays_in_its_dimensions():
    lens = [130]
    tables, nb = tables_of(lens, 64, 4)
    pages = Pages(7, nb, 64, 1, 128)
    ref, size = _reference(rng_rows(1, (1, 2, 128), "bf16"), pages, tables, [1], lens, 128 ** -0.5)
    pages.np[1][1][tables[0][1], 0, 2, 5] = np.nan     # group 2 of one token's value
    out = paged_decode(rng_rows(1, (1, 2, 128), "bf16").cuda(), *pages.gpu(), _int(lens),
                       _int(tables), None).cpu()
    assert torch.isnan(out[..., 64:96]).all()
    keep = [d for d in range(128) if not 64 <= d < 96]
    assert_close(out[..., keep], ref[..., keep], size[..., keep], "bf16", "fp4 NaN value")


def test_scores_far_apart_and_scales_of_many_magnitudes():
    """One key far above the others, values from 1e-3 to 1e3: the running maximum moves late."""
    n, hkv, d = 700, 2, 128
    rows_k = rng_rows(1, (n, hkv, d), "bf16").double().numpy()
    rows_k[650] *= 60
    rows_k[10] *= -40
    rows_v = rng_rows(2, (n, hkv, d), "bf16", spread=1e3).double().numpy()
    nb, bs = 11, 64
    pages = Pages(3, nb, bs, hkv, d)
    for i, rows in enumerate((rows_k, rows_v)):
        orc.store(rows, *pages.np[i], np.arange(n), i == 0)
    q = rng_rows(5, (1, 4, d), "bf16").cuda()
    out = paged_decode(q, *pages.gpu(), _int([n]), _int([np.arange(nb)]), None)
    ref, size = _reference(q, pages, [np.arange(nb)], [1], [n], d ** -0.5)
    assert_close(out, ref, size, "bf16", "fp4 far scores")


def test_page_ids_outside_the_cache_are_not_followed():
    lens = [100, 100, 100]
    tables, nb = tables_of(lens, 64, 4)
    pages = Pages(7, nb, 64, 2, 128)
    q = rng_rows(1, (3, 4, 128), "bf16").cuda()
    ref, size = _reference(q, pages, tables, [1] * 3, lens, 128 ** -0.5)
    bad = tables.copy()
    bad[1] = [nb, -7]
    out = paged_decode(q, *pages.gpu(), _int(lens), _int(bad), None)
    assert torch.isfinite(out).all()
    for b in (0, 2):
        assert_close(out[b], ref[b], size[b], "bf16", "fp4 beside a bad table")
    # lengths beyond the table's pages are cut to them
    out = paged_decode(q, *pages.gpu(), _int([10 ** 6] * 3), _int(tables), None)
    full, fsize = _reference(q, pages, tables, [1] * 3, [128] * 3, 128 ** -0.5)
    assert_close(out, full, fsize, "bf16", "fp4 lengths past the table")


def test_without_a_block_table_every_sequence_is_a_page():
    lens = [5, 48]
    pages = Pages(7, 2, 48, 2, 128)
    q = rng_rows(1, (2, 1, 4, 128), "bf16").cuda()
    out = flash_attn_with_kvcache(q, *pages.gpu(), cache_seqlens=_int(lens), causal=True)
    ref, size = _reference(q[:, 0], pages, [[0], [1]], [1, 1], lens, 128 ** -0.5)
    assert_close(out[:, 0], ref, size, "bf16", "fp4 no table")
    out = flash_attn_with_kvcache(q, *pages.gpu(), cache_seqlens=7, causal=True)
    ref, size = _reference(q[:, 0], pages, [[0], [1]], [1, 1], [7, 7], 128 ** -0.5)
    assert_close(out[:, 0], ref, size, "bf16", "fp4 int length")


def test_pages_past_4_gib():
    hkv, d, bs = 8, 128, 256
    nb = (1 << 32) // (hkv * bs * d // 2) + 4
    small = Pages(7, 4, bs, hkv, d)
    kc, vc = Fp4Cache.zeros(nb, bs, hkv, d), Fp4Cache.zeros(nb, bs, hkv, d)
    for c, s in zip((kc, vc), small.gpu()):
        c.data[-4:], c.scale[-4:] = s.data, s.scale
    lens = [1000, 3]
    tables = np.array([[1, 3, 0, 2], [2, -1, -1, -1]], np.int32)
    q = rng_rows(1, (2, 16, d), "bf16").cuda()
    say("fp4 decode past 4 GiB")
    out = paged_decode(q, kc, vc, _int(lens), _int(np.where(tables >= 0, tables + nb - 4, -1)), None)
    ref, size = _reference(q, small, tables, [1, 1], lens, d ** -0.5)
    assert_close(out, ref, size, "bf16", "fp4 past 4 GiB")


def test_a_captured_decode_follows_its_inputs():
    """A graph replayed with other lengths, tables and queries, eager calls between the replays."""
    bs, hkv, hq, d = 256, 8, 16, 128
    first = [300, 40, 0, 700]
    tables, nb = tables_of([700] * 4, bs, 3)
    pages = Pages(7, nb, bs, hkv, d)
    kc, vc = pages.gpu()
    q, lens, bt = rng_rows(1, (4, hq, d), "bf16").cuda(), _int(first), _int(tables)
    paged_decode(q, kc, vc, lens, bt, None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_decode(q, kc, vc, lens, bt, None)
    for i, now in enumerate([first, [1, 2, 3, 4], [700, 0, 256, 257], first]):
        q.copy_(rng_rows(20 + i, (4, hq, d), "bf16"))
        lens.copy_(_int(now))
        graph.replay()
        eager = paged_decode(q, kc, vc, lens, bt, None)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        ref, size = _reference(q, pages, tables, [1] * 4, now, d ** -0.5)
        assert_close(out, ref, size, "bf16", f"fp4 replay {i}")


def test_two_streams_at_once():
    lens = [900] * 8
    tables, nb = tables_of(lens, 256, 3)
    pages = Pages(7, nb, 256, 8, 128)
    kc, vc = pages.gpu()
    qs = [rng_rows(i, (8, 16, 128), "bf16").cuda() for i in range(2)]
    args = (_int(lens), _int(tables), None)
    want = [paged_decode(q, kc, vc, *args) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_decode(qs[i], kc, vc, *args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_refusals():
    pages = Pages(7, 2, 64, 2, 128)
    kc, vc = pages.gpu()
    q = rng_rows(1, (2, 4, 128), "bf16").cuda()
    lens, bt = _int([3, 4]), _int([[0], [1]])
    for bad in (lambda: paged_decode(q, kc, vc, lens, bt[:1], None),
                lambda: paged_decode(q, kc, vc, lens[:1], bt, None),
                lambda: paged_decode(q[..., :64], kc, vc, lens, bt, None),
                lambda: paged_decode(q.float(), kc, vc, lens, bt, None),
                lambda: paged_decode(q[:, :3], kc, vc, lens, bt, None),
                lambda: paged_decode(q, kc, vc, lens, bt, 0.0),
                lambda: paged_decode(q, kc, vc, lens, bt, None, out=q.float()),
                lambda: paged_decode(q, kc, pages.np[1], lens, bt, None),
                lambda: varlen_prefill(q, kc, vc, _int([0, 2]), _int([0, 3, 4]), 2, None,
                                       block_table=bt[:1])):
        with pytest.raises(Exception) as e:
            bad()
        assert "Nvk" in type(e.value).__name__
    with pytest.raises(NotImplementedError):
        flash_attn_with_kvcache(q.view(1, 2, 4, 128), kc, vc, cache_seqlens=_int([3]),
                                block_table=_int([[0]]))
