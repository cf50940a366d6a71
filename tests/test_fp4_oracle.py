"""The 4-bit cache on the CPU: the oracle's format against brute force, the cache type and every
refusal that needs no GPU."""
import numpy as np
import pytest
import torch

from nanovllm_amd import Fp4Cache, _lib, load_kvcache, store_kvcache
from nanovllm_amd.flash_api import flash_attn_with_kvcache, paged_decode, varlen_prefill
from oracle import fp4_oracle as orc


def test_codes_are_the_nearest_and_ties_go_to_the_even_code():
    # scale 1 (largest magnitude 6): all borders and values between them
    x = np.zeros(32)
    x[:16] = [6, 0.25, 0.2501, 0.75, 0.7499, 1.25, 1.2501, 1.75, 1.7499, 2.5, 2.501, 3.5, 3.499, 5,
              5.001, -5]
    codes, scale = orc.quantise(x)
    assert scale == np.float16(1)
    assert codes[:16].tolist() == [7, 0, 1, 2, 1, 2, 3, 4, 3, 4, 5, 6, 5, 6, 7, 14]
    assert not codes[16:].any()


def test_round_trip_is_within_half_a_step_of_the_grid():
    rng = np.random.default_rng(0)
    for d in (64, 128):
        rows = rng.standard_normal((40, 3, d)).astype(np.float16).astype(np.float64)
        data = np.zeros((4, 3, 16, d // 2), np.uint8)
        scale = np.zeros((4, 3, d // 32, 16), np.float16)
        slots = rng.permutation(64)[:40]
        for keys in (True, False):
            orc.store(rows, data, scale, slots, keys)
            got = orc.values(data, scale, keys).reshape(64, 3, d)[slots]
            s = scale.swapaxes(-1, -2).astype(np.float64).swapaxes(1, 2).reshape(64, 3, -1)[slots]
            # the widest gap is 2 (from 4 to 6); the scale's own rounding moves the top by 6 * 2^-11
            assert (np.abs(got - rows) <= s.repeat(32, -1) * (1 + 6 * 2.0 ** -11)).all()


def test_key_rows_are_a_permutation_of_units_of_eight():
    for d in (64, 128):
        p = orc.places(d, True)
        assert sorted(p) == list(range(d))
        assert (p.reshape(-1, 8) == p.reshape(-1, 8)[:, :1] + np.arange(8)).all()
        # the group of a place: unit (D / 32) g + s belongs to group s
        assert ((p // 8) % (d // 32) == np.arange(d) // 32).all()


def test_groups_without_a_scale_and_groups_that_are_not_finite():
    x = np.zeros((4, 32))
    x[1, 3] = -(2.0 ** -23)           # / 6 rounds to 0 in f16
    x[2, 0], x[2, 1] = np.inf, 1.0
    x[3, 31] = np.nan
    codes, scale = orc.quantise(x)
    assert scale[:2].tolist() == [[0], [0]] and np.isnan(scale[2:]).all()
    assert not codes[0].any() and not codes[2:].any() and codes[1].tolist().count(8) == 1


def _caches(nb=2, h=2, bs=16, d=128):
    return Fp4Cache.zeros(nb, bs, h, d, device="cpu"), Fp4Cache.zeros(nb, bs, h, d, device="cpu")


def test_cache_type():
    kc, vc = _caches(3, 2, 32, 64)
    assert kc.data.shape == (3, 2, 32, 32) and kc.data.dtype == torch.uint8
    assert kc.scale.shape == (3, 2, 2, 32) and kc.scale.dtype == torch.float16
    assert kc.numel() == 3 * 2 * 32 * 64
    assert Fp4Cache.zeros(0, 256, 8, 128, device="cpu").numel() == 0
    for bad in ((2, 8, 2, 128), (2, 0, 2, 128), (2, 24, 2, 128), (2, 16, 2, 96)):
        with pytest.raises(_lib.NvkError):
            Fp4Cache.zeros(*bad, device="cpu")


def test_cpu_tensors_are_refused():
    kc, vc = _caches()
    rows = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    slots = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: store_kvcache(rows, rows, kc, vc, slots),
                 lambda: load_kvcache(kc, vc, slots),
                 lambda: paged_decode(rows, kc, vc, slots, slots.view(4, 1), None),
                 lambda: flash_attn_with_kvcache(rows[:, None], kc, vc, cache_seqlens=slots,
                                                 block_table=slots.view(4, 1))):
        with pytest.raises(_lib.NvkError, match="CPU tensor"):
            call()


def test_caches_that_do_not_fit_are_refused():
    kc, vc = _caches()
    rows = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    slots = torch.zeros(4, dtype=torch.int32)
    plain = torch.zeros(2, 16, 2, 128, dtype=torch.bfloat16)
    other = Fp4Cache.zeros(3, 16, 2, 128, device="cpu")
    for k, v in ((kc, plain), (plain, vc), (kc, other), (kc, Fp4Cache(vc.data, vc.scale.float())),
                 (kc, Fp4Cache(vc.data[:, :, ::2], vc.scale)),
                 (kc, Fp4Cache(vc.data, vc.scale.transpose(-1, -2)))):
        for call in (lambda: store_kvcache(rows, rows, k, v, slots),
                     lambda: load_kvcache(k, v, slots),
                     lambda: paged_decode(rows, k, v, slots, slots.view(4, 1), None)):
            with pytest.raises(_lib.NvkError):
                call()
    with pytest.raises(_lib.NvkError, match="block_table"):
        varlen_prefill(rows, kc, vc, slots[:2], slots[:2], 4, None)
    with pytest.raises(_lib.NvkError, match="bfloat16 and float16"):
        store_kvcache(rows.float(), rows.float(), kc, vc, slots)
    with pytest.raises(_lib.NvkError, match="bfloat16 and float16"):
        load_kvcache(kc, vc, slots, torch.float32)
    with pytest.raises(AssertionError):
        store_kvcache(rows[:, :1], rows[:, :1], kc, vc, slots)      # another head count
    with pytest.raises(AssertionError):
        store_kvcache(rows, rows, kc, vc, slots[:3])


@pytest.mark.skipif(torch.cuda.is_available(),
                    reason="passes fake device pointers; a validation regression must not be "
                           "able to launch a kernel on them, so it only runs without a GPU")
def test_error_codes_without_launching():
    lib = _lib.load()
    EINVAL, EUNSUPPORTED, EALIGN, EWORKSPACE = -1, -2, -3, -4
    # key, stride, value, stride, k data, k scale, v data, v scale, slots, n, hkv, d, bs, nb, dtype
    st = [16, 1024, 16, 1024, 16, 16, 16, 16, 16, 4, 8, 128, 256, 4, 0, None]
    change = lambda args, **kw: [kw.get(f"a{i}", x) for i, x in enumerate(args)]
    assert lib.nvk_fp4_store(*change(st, a9=0)) == 0
    assert lib.nvk_fp4_store(*change(st, a9=-1)) == EINVAL
    assert lib.nvk_fp4_store(*change(st, a0=None)) == EINVAL
    assert lib.nvk_fp4_store(*change(st, a1=1016)) == EINVAL          # rows overlap
    assert lib.nvk_fp4_store(*change(st, a11=96)) == EUNSUPPORTED
    assert lib.nvk_fp4_store(*change(st, a12=24)) == EUNSUPPORTED
    assert lib.nvk_fp4_store(*change(st, a14=2)) == EUNSUPPORTED      # f32 rows
    assert lib.nvk_fp4_store(*change(st, a0=24)) == EALIGN
    assert lib.nvk_fp4_store(*change(st, a3=1028)) == EALIGN
    assert lib.nvk_fp4_store(*change(st, a5=24)) == EALIGN
    ld = [16, 16, 16, 16, 16, 4, 8, 128, 256, 4, 16, 1024, 16, 1024, 0, None]
    assert lib.nvk_fp4_load(*change(ld, a5=0)) == 0
    assert lib.nvk_fp4_load(*change(ld, a10=None)) == EINVAL
    assert lib.nvk_fp4_load(*change(ld, a14=2)) == EUNSUPPORTED
    assert lib.nvk_fp4_load(*change(ld, a12=8)) == EALIGN
    # q, strides, total_q, caches, cu_q, seqlens, batch, max_q, max_k, table, stride, width, bs,
    # nb, hq, hkv, d, scale, out, strides, workspace, bytes, dtype, stream
    need = lib.nvk_fp4_attention_workspace_size(2, 1, 0, 16, 8, 128, 256, 8)
    assert need > 0
    at = [16, 2048, 128, 2, 16, 16, 16, 16, None, 16, 2, 1, 0, 16, 8, 8, 256, 64, 16, 8, 128, 0.1, 16,
          2048, 128, 256, need, 0, None]
    assert lib.nvk_fp4_attention(*change(at, a3=0, a10=0)) == 0
    assert lib.nvk_fp4_attention(*change(at, a3=3)) == EINVAL         # 2 sequences, 3 queries
    assert lib.nvk_fp4_attention(*change(at, a21=0.0)) == EINVAL
    assert lib.nvk_fp4_attention(*change(at, a12=-1)) == EINVAL
    assert lib.nvk_fp4_attention(*change(at, a18=12)) == EINVAL       # 12 % 8
    assert lib.nvk_fp4_attention(*change(at, a14=4)) == EINVAL        # tables overlap
    assert lib.nvk_fp4_attention(*change(at, a9=None)) == EINVAL
    assert lib.nvk_fp4_attention(*change(at, a20=96)) == EUNSUPPORTED
    assert lib.nvk_fp4_attention(*change(at, a16=8)) == EUNSUPPORTED
    assert lib.nvk_fp4_attention(*change(at, a17=0)) == EUNSUPPORTED  # no page
    assert lib.nvk_fp4_attention(*change(at, a18=256)) == EUNSUPPORTED  # 32 heads per kv head
    assert lib.nvk_fp4_attention(*change(at, a27=2)) == EUNSUPPORTED
    assert lib.nvk_fp4_attention(*change(at, a0=8)) == EALIGN
    assert lib.nvk_fp4_attention(*change(at, a2=132)) == EALIGN
    assert lib.nvk_fp4_attention(*change(at, a22=20)) == EALIGN
    assert lib.nvk_fp4_attention(*change(at, a25=None)) == EWORKSPACE
    assert lib.nvk_fp4_attention(*change(at, a26=need - 1)) == EWORKSPACE
    assert lib.nvk_fp4_attention(*change(at, a25=128)) == EALIGN
    size = lib.nvk_fp4_attention_workspace_size
    assert size(2049, 1, 0, 16, 8, 128, 256, 8) == 0 and size(2, 1, 0, 16, 8, 128, 24, 8) == 0
    assert size(2, 0, 0, 16, 8, 128, 256, 8) == 0 and size(2, 1, 0, 16, 5, 128, 256, 8) == 0
    assert size(2048, 4096, 0, 16, 1, 128, 256, 1 << 20) == 0         # past 32-bit work counts
    # many queries: f16 pages of the keys, 512 MiB of them or one sequence's, and no more with a
    # bound on the keys
    assert size(1, 1000, 9300, 16, 8, 128, 256, 64) > 2 * 37 * 256 * 8 * 128 * 2
    assert size(1, 1000, 9300, 16, 8, 128, 256, 64) < size(1, 1000, 0, 16, 8, 128, 256, 64)
    assert size(64, 1000, 9300, 16, 8, 128, 256, 64) < 700 << 20
