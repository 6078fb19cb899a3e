"""A ragged batch over a paged cache of 8-bit codes, and what its codes stand for in 64 bits (tqhip_kv_cache8), for the tests of the calls that
write and read it."""
import numpy as np
import torch

from batch_ref import Batch

I8, E4M3 = 3, 4
TOP = {I8: 127.0, E4M3: 448.0}
LEAST = np.float32(2.0 ** -60)


def to_codes(x, dtype):
    """float32 -> codes (uint8), rounded to nearest even."""
    x = np.clip(np.asarray(x, np.float32), -TOP[dtype], TOP[dtype])
    if dtype == I8:
        return np.rint(x).astype(np.int8).view(np.uint8)
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def from_codes(codes, dtype):
    """uint8 -> float64."""
    if dtype == I8:
        return codes.view(np.int8).astype(np.float64)
    return torch.from_numpy(np.ascontiguousarray(codes)).view(torch.float8_e4m3fn).double().numpy()


class Values:
    """What Batch's forms look at: `values` in float64."""

    def __init__(self, values):
        self.values = values


class Batch8(Batch):
    """Batch with its rows quantized: scales of `spread` random powers around the rows' own, rows that no position uses hold garbage (NaN where
    the type has it), blocks without a used row scales of NaN. `scales` is [page][head][block][2] float32, `codes` [2][page][row][head][dim]."""

    def __init__(self, tq, new, kv, page, Hk, D, dtype, block=None, seed=0, spread=1.0, **kw):
        super().__init__(tq, new, kv, page, Hk, D, 0, seed=seed, **kw)
        self.dtype, self.block = dtype, block or page
        assert page % self.block == 0
        self.n_blocks = page // self.block
        x = np.stack([self.rows(self.k.values), self.rows(self.v.values)])  # [2][page][row][head][dim], NaN where no position is
        self.used = ~np.isnan(x[0, :, :, 0, 0])
        per = np.abs(x).reshape(2, self.n_pages, self.n_blocks, self.block, Hk, D)
        top = np.nanmax(np.where(np.isnan(per), 0.0, per), axis=(3, 5))  # [2][page][block][head]
        scale = (top / TOP[dtype] * 2.0 ** self.rng.uniform(0, spread, top.shape)).astype(np.float32)
        scale[scale == 0] = np.nan
        self.scales = np.ascontiguousarray(scale.transpose(1, 3, 2, 0))
        by = np.repeat(scale, self.block, axis=2)[..., None]  # [2][page][row][head][1]
        with np.errstate(invalid="ignore"):
            self.codes = to_codes(np.where(np.isnan(x / by), 0.0, x / by), dtype)
        junk = self.rng.integers(0, 256, self.codes.shape).astype(np.uint8)
        if dtype == E4M3:
            junk[..., ::3] = 0x7f
        self.codes = np.where(self.used[None, :, :, None, None], self.codes, junk)
        self.put()

    def put(self):
        """To the device, and the values that it all stands for."""
        lay = self.codes.transpose(0, 1, 3, 2, 4) if self.layout == "head" else self.codes
        self.d_codes = self.tq.DeviceBuffer.from_array(np.ascontiguousarray(lay))
        self.d_scales = self.tq.DeviceBuffer.from_array(self.scales)
        self.stand_for()
        size = self.codes[0].size
        strides = dict(page_stride=self.page * self.Hk * self.D, token_stride=self.D, head_stride=self.page * self.D) if self.layout == "head" else {}
        self.c = self.tq.KvCache8(k=self.d_codes.ptr, v=self.d_codes.ptr + size, scales=self.d_scales.ptr, dtype=self.dtype, n_pages=self.n_pages,
                                  page_size=self.page, block=self.block, n_kv_heads=self.Hk, head_dim=self.D, **strides)

    def stand_for(self):
        by = np.repeat(self.scales.astype(np.float64).transpose(3, 0, 2, 1), self.block, axis=2)[..., None]
        with np.errstate(invalid="ignore"):
            x = from_codes(self.codes, self.dtype) * by
        self.k, self.v = (Values(y.transpose(0, 2, 1, 3) if self.layout == "head" else y) for y in x)

    def read(self):
        """What the device holds now."""
        shape = self.codes.transpose(0, 1, 3, 2, 4).shape if self.layout == "head" else self.codes.shape
        codes = self.d_codes.download(np.uint8, self.codes.size).reshape(shape)
        self.codes = codes.transpose(0, 1, 3, 2, 4).copy() if self.layout == "head" else codes
        self.scales = self.d_scales.download(np.float32, self.scales.size).reshape(self.scales.shape)
        self.stand_for()
        return self
