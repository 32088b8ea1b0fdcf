"""Ragged batches over pages of 8 bits for the tests, and how a row is held, in 64 bits (CPU)."""

import math

import torch

import paged_ref as R

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def exponent(rows):
    """The least e from -15 to 7 with |x| <= 448 * 2^e for a row's largest finite x."""
    most = torch.where(rows.isfinite(), rows, 0.0).abs().amax(-1).double()
    e = torch.full(most.shape, -15, dtype=torch.int64)
    for i in range(-15, 7):
        e[most > 448.0 * 2.0 ** i] = i + 1
    return e


def hold(rows):
    """(codes, exponents + 127 as bytes, the values that these stand for) of rows [..., dim]."""
    e = exponent(rows)
    x = torch.where(rows.isfinite(), rows, math.nan).double() * 2.0 ** -e.double()[..., None]
    codes = x.clamp(-448.0, 448.0).float().to(E4M3)
    return codes, (e + 127).to(torch.uint8), codes.float() * torch.exp2(e.float())[..., None]


class Batch8(R.Batch):
    """R.Batch whose keys and values are what pages of 8 bits hold: `k`, `v` are those values, unused rows hold codes of
    NaN and any exponent."""

    def __init__(self, *args, sizes=True, **kw):
        super().__init__(*args, **kw)
        g = torch.Generator().manual_seed(kw.get("seed", 0) + 1)
        shape = (self.pages, self.nkv, self.page, self.dim)
        for name in ("k", "v"):
            codes = torch.full(shape, 0x7f, dtype=torch.uint8)
            scale = torch.randint(0, 256, shape[:3], generator=g).to(torch.uint8)
            rows = []
            for i, (_, kv) in enumerate(self.spec):
                x = getattr(self, name)[i].float()
                if sizes:  # rows of sizes from 1/8 to 8 times
                    x = x * torch.exp2(torch.randint(-3, 4, x.shape[:2], generator=g).float())[..., None]
                c, e, held = hold(x)
                rows.append(held)
                for p in range(kv):
                    at = int(self.table[i, p // self.page]), slice(None), p % self.page
                    codes[at], scale[at] = c[p].view(torch.uint8), e[p]
            setattr(self, name, rows)
            setattr(self, name + "_pages", codes.view(E4M3))
            setattr(self, name + "_scale", scale.view(E8M0))
