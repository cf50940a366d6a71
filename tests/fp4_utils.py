"""Helpers of the 4-bit cache's tests (not collected by pytest)."""
import numpy as np
import torch

from nanovllm_amd import Fp4Cache
from oracle import fp4_oracle as orc

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}     # eps / 2


def rng_rows(seed, shape, dtype, spread=1.0):
    """N(0, 1) rows, each row and head times a magnitude of its own where spread > 1."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    if spread != 1.0:
        x *= spread ** (2 * torch.rand(*shape[:-1], 1, generator=gen) - 1)
    return x.to(DTYPES[dtype])


class Pages:
    """A pair of 4-bit caches in numpy and on the GPU, filled with N(0, 1) rows."""

    def __init__(self, seed, num_blocks, block_size, hkv, d, dtype="bf16"):
        self.nb, self.bs, self.hkv, self.d = num_blocks, block_size, hkv, d
        self.np = []
        for i in range(2):
            rows = rng_rows(seed + i, (num_blocks, hkv, block_size, d), dtype).double().numpy()
            codes, scale = orc.quantise(rows)
            self.np.append((orc.pack(codes, i == 0), np.swapaxes(scale, -1, -2).copy()))

    def gpu(self):
        return [Fp4Cache(torch.from_numpy(a).cuda(), torch.from_numpy(s).cuda())
                for a, s in self.np]

    def values(self, i):
        return orc.values(*self.np[i], keys=i == 0)

    def rows(self, table, n):
        """Keys and values [n, Hkv, D] of a block table's first n slots."""
        p = np.arange(n)
        at = (np.asarray(table)[p // self.bs], p % self.bs)
        return self.values(0)[at], self.values(1)[at]


def tables_of(lens, block_size, seed, pages=None):
    """(tables padded with -1 [B, W] int32, pages needed): shuffled, unshared pages."""
    need = [max(0, -(-n // block_size)) for n in lens]
    total = max(1, sum(need))
    ids = np.random.default_rng(seed).permutation(total)
    width = max(1, max(need))
    out = np.full((len(lens), width), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        out[b, :n] = ids[at:at + n]
        at += n
    return out, total


def assert_close(out, ref, size, dtype, what):
    """|out - ref| <= half a step of the output's type + `size` (see oracle.fp4_oracle.attention)."""
    got = out.detach().double().cpu().numpy().reshape(ref.shape)
    tol = HALF_STEP[dtype] * (np.abs(ref) + size) + size + 2.0 ** -25
    bad = ~(np.abs(got - ref) <= tol)
    assert not bad.any(), (f"{what}: {bad.sum()} of {bad.size} beyond the bound, worst "
                           f"{np.nanmax(np.abs(got - ref) / tol):.2f} of it at {np.argwhere(bad)[:3]}")
