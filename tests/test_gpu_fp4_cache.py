"""The 4-bit cache as it is written and read back, on the GPU: bytes and scales equal to the
oracle's, values rounded once."""
import numpy as np
import pytest
import torch

from fp4_utils import DTYPES, Pages, rng_rows
from gpu_utils import say
from nanovllm_amd import Fp4Cache, load_kvcache, store_kvcache
from oracle import fp4_oracle as orc

pytestmark = pytest.mark.gpu


def _numpy(c):
    return c.data.cpu().numpy(), c.scale.cpu().numpy()


def _store_and_check(key, value, slots, nb, bs, seed, what):
    """Stores into caches that hold something already and compares every byte."""
    hkv, d = key.shape[1:]
    pages = Pages(seed, nb, bs, hkv, d)
    gpu = pages.gpu()
    say(what)
    store_kvcache(key, value, *gpu, slots)
    torch.cuda.synchronize()
    for i, rows in enumerate((key, value)):
        data, scale = pages.np[i][0].copy(), pages.np[i][1].copy()
        orc.store(rows.double().cpu().numpy(), data, scale, slots.cpu().numpy(), i == 0)
        got_d, got_s = _numpy(gpu[i])
        np.testing.assert_array_equal(got_s.view(np.uint16), scale.view(np.uint16), err_msg=what)
        np.testing.assert_array_equal(got_d, data, err_msg=what)
    return gpu


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hkv,d,bs", [(8, 128, 256), (2, 64, 16), (5, 128, 48), (1, 128, 64)])
@pytest.mark.parametrize("n", [1, 7, 300])
def test_store_writes_what_the_format_says(n, hkv, d, bs, dtype):
    nb = -(-n // bs) + 3
    gen = np.random.default_rng(n)
    slots = gen.permutation(nb * bs)[:n].astype(np.int32)
    slots[gen.permutation(n)[:n // 5]] = -1
    key, value = (rng_rows(10 * n + i, (n, hkv, d), dtype, spread=1e3).cuda() for i in range(2))
    _store_and_check(key, value, torch.from_numpy(slots).cuda(), nb, bs, n, f"fp4 store {n} {dtype}")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_store_of_consecutive_slots(dtype):
    """A prompt's tokens: runs of slots that start and end anywhere in a page."""
    n, hkv, d, bs = 211, 2, 128, 64
    slots = (np.arange(n) + 5).astype(np.int32)
    key, value = (rng_rows(i, (n, hkv, d), dtype).cuda() for i in range(2))
    _store_and_check(key, value, torch.from_numpy(slots).cuda(), 4, bs, 3, f"fp4 store run {dtype}")


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_store_of_borders_and_odd_values(dtype):
    """Every border between codes at scales of every exponent (exact ties), zeros of both signs,
    subnormal numbers, the largest ones, infinities and NaN."""
    t = DTYPES[dtype]
    borders = torch.tensor([6, .25, -.25, .75, -.75, 1.25, -1.25, 1.75, -1.75, 2.5, -2.5, 3.5, -3.5,
                            5, -5, .5, -1, 1.5, -2, 3, -4, -6, 0, -0.0, .125, 4.5, -5.5, 2.25, .3,
                            -.3, 1., .9])
    top = torch.finfo(t).max
    lo, hi = (-24, 13) if dtype == "fp16" else (-40, 30)
    rows = [borders * 2.0 ** e for e in range(lo, hi)]
    # scales with all bits set, times each border: ties at products of 13 bits are not 16-bit values,
    # their neighbours are
    rows += [borders * (1 + i / 64) for i in range(64)]
    odd = torch.zeros(8, 32)
    odd[0, 5] = top
    odd[1, :] = -top
    odd[2, 31] = float("inf")
    odd[3, 0] = float("nan")
    odd[4, 7], odd[4, 8] = float("-inf"), float("nan")
    odd[5, 2] = torch.finfo(t).tiny
    odd[6, 2], odd[6, 3] = torch.finfo(t).smallest_normal / 4, -1e-30
    odd[7, :16] = -0.0
    x = torch.cat([torch.stack(rows).to(t), odd.to(t)])
    x = x[: len(x) // 4 * 4].reshape(-1, 1, 128)
    slots = torch.arange(len(x), dtype=torch.int32).cuda()
    _store_and_check(x.cuda(), x.flip(0).cuda(), slots, -(-len(x) // 16), 16, 7,
                     f"fp4 store borders {dtype}")


def test_store_of_a_packed_projection_and_slots_outside():
    n, hkv, d = 50, 4, 128
    qkv = rng_rows(1, (n, 16 * d), "bf16").cuda()
    key, value = qkv[:, 8 * d:12 * d].view(n, hkv, d), qkv[:, 12 * d:].view(n, hkv, d)
    slots = torch.arange(n, dtype=torch.int64).cuda() * 3 - 10     # some below 0, some past the end
    before = qkv.clone()
    _store_and_check(key, value, slots, 6, 16, 2, "fp4 store packed, slots outside")
    assert torch.equal(qkv, before)


def test_nothing_is_stored_for_no_tokens():
    kc, vc = Fp4Cache.zeros(2, 16, 2, 128), Fp4Cache.zeros(2, 16, 2, 128)
    empty = torch.empty(0, 2, 128, dtype=torch.bfloat16, device="cuda")
    slots = torch.empty(0, dtype=torch.int32, device="cuda")
    store_kvcache(empty, empty, kc, vc, slots)
    k, v = load_kvcache(kc, vc, slots)
    assert k.shape == v.shape == (0, 2, 128) and not kc.data.any()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("hkv,d,bs", [(8, 128, 256), (2, 64, 16), (5, 128, 48)])
@pytest.mark.parametrize("n", [1, 33, 500])
def test_load_gives_the_values_rounded_once(n, hkv, d, bs, dtype):
    nb = -(-n // bs) + 2
    pages = Pages(n, nb, bs, hkv, d, dtype)
    slots = np.random.default_rng(n).permutation(nb * bs)[:n].astype(np.int32)
    slots[::7] = -1
    if n > 1:
        slots[1], slots[2] = nb * bs, slots[3]       # past the end; the same slot twice
    say(f"fp4 load {n} x {hkv} x {d} {dtype}")
    got = load_kvcache(*pages.gpu(), torch.from_numpy(slots).cuda(), DTYPES[dtype])
    for i in range(2):
        v = pages.values(i).reshape(nb * bs, hkv, d)
        ok = ((slots >= 0) & (slots < nb * bs))[:, None, None]
        want = np.where(ok, v[np.clip(slots, 0, nb * bs - 1)], 0.0)
        want = torch.from_numpy(want).float().to(DTYPES[dtype])       # exact in f32, then one rounding
        assert torch.equal(got[i].cpu(), want)


def test_load_of_what_was_not_finite():
    kc, vc = Fp4Cache.zeros(1, 16, 1, 64), Fp4Cache.zeros(1, 16, 1, 64)
    x = torch.ones(2, 1, 64, dtype=torch.float16, device="cuda")
    x[1, 0, 40] = float("inf")
    slots = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    store_kvcache(x, x, kc, vc, slots)
    for got in load_kvcache(kc, vc, slots, torch.float16):
        assert torch.isnan(got[1, 0, 32:]).all() and torch.isfinite(got[1, 0, :32]).all()
        assert torch.isfinite(got[0]).all()


def test_offsets_past_32_bits():
    """Pages beyond 2^32 bytes of codes."""
    hkv, d, bs = 8, 128, 256
    nb = (1 << 32) // (hkv * bs * d // 2) + 8
    kc, vc = Fp4Cache.zeros(nb, bs, hkv, d), Fp4Cache.zeros(nb, bs, hkv, d)
    slots = torch.tensor([0, 17, (nb - 1) * bs + 255, (nb - 8) * bs], dtype=torch.int32,
                         device="cuda")
    key, value = (rng_rows(i, (4, hkv, d), "bf16").cuda() for i in range(2))
    say("fp4 store and load past 4 GiB")
    store_kvcache(key, value, kc, vc, slots)
    k, v = load_kvcache(kc, vc, slots)
    for rows, got in ((key, k), (value, v)):
        codes, scale = orc.quantise(rows.double().cpu().numpy())
        want = orc.MAGNITUDES[codes & 7] * np.where(codes & 8, -1, 1) \
            * scale.astype(np.float64).repeat(32, -1)
        assert torch.equal(got.cpu(), torch.from_numpy(want).float().to(torch.bfloat16))
    assert int(kc.data[1:nb - 8].count_nonzero()) == 0


def test_more_tokens_than_one_grid_dimension_holds():
    """More than 32768 pieces of 16 tokens: the same as two calls of fewer."""
    n, d, bs = 16 * 32768 + 1000, 128, 256
    gen = torch.Generator(device="cuda").manual_seed(3)
    key, value = torch.randn(2, n, 1, d, generator=gen, device="cuda").to(torch.bfloat16)
    slots = torch.arange(n, dtype=torch.int32, device="cuda").flip(0)
    once, twice = ([Fp4Cache.zeros(-(-n // bs), bs, 1, d) for _ in range(2)] for _ in range(2))
    say("fp4 store and load of 525288 tokens")
    store_kvcache(key, value, *once, slots)
    half = n // 2
    for part in (slice(0, half), slice(half, n)):
        store_kvcache(key[part], value[part], *twice, slots[part])
    rows = load_kvcache(*once, slots)
    for i in range(2):
        assert torch.equal(once[i].data, twice[i].data)
        assert torch.equal(once[i].scale, twice[i].scale)
        parts = [load_kvcache(*once, slots[part])[i] for part in (slice(0, half), slice(half, n))]
        assert torch.equal(rows[i], torch.cat(parts))
