"""Plain implementations of the operators in 4-bit floating point, and a paged cache with shuffled pages."""

from __future__ import annotations

import torch

from deterministic_inference_b200.kernels import ops
from tests.int8_util import Int8Case

FLOOR = 2.0 ** -100
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantised(x: torch.Tensor):
    """Codes (uint8 [.., ceil(K / 2)]), block scales (float8_e4m3fn), exponent bytes of the last axis' rows, with the float32
    operations that define them; a code by comparison with the borders between the codes."""
    x = x.float()
    k = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -k % 16)).unflatten(-1, (-1, 16))
    tops = x.abs().amax(-1)
    a = tops.amax(-1)
    bad = ~torch.isfinite(a)
    share, e = torch.frexp(torch.where(bad, torch.ones_like(a), a).clamp(min=FLOOR))
    e = e - 12 + (share > 2688 / 4096)
    down = torch.ldexp(torch.ones_like(a), -e)[..., None]
    scales = (torch.where(bad[..., None], torch.zeros_like(tops), tops) * down / torch.full_like(tops, 6.0)).to(torch.float8_e4m3fn)
    b = scales.float()[..., None]
    y = torch.where((b > 0) & ~bad[..., None, None], x * down[..., None] / b, torch.zeros_like(x))
    code = torch.zeros_like(y, dtype=torch.uint8)
    # a border belongs to the code whose last bit is zero: the upper one where that is even
    for border, upper in ((0.25, 1), (0.75, 2), (1.25, 3), (1.75, 4), (2.5, 5), (3.5, 6), (5.0, 7)):
        code += (y.abs() >= border if upper % 2 == 0 else y.abs() > border).to(torch.uint8)
    code += torch.signbit(y).to(torch.uint8) * 8
    code = code.flatten(-2)[..., :k + k % 2]
    if k % 2:
        code[..., -1] = 0
    packed = code[..., ::2] + code[..., 1::2] * 16
    return packed, scales, torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)


def values(codes, scales, exponents, k: int, dtype=torch.float64) -> torch.Tensor:
    """What such rows stand for."""
    table = torch.cat([E2M1, -E2M1]).to(codes.device, dtype)
    y = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()][..., :k]
    unit = torch.where(exponents == 255, torch.nan, torch.exp2(exponents.to(dtype) - 127))
    return y * scales.to(dtype).repeat_interleave(16, -1)[..., :k] * unit[..., None]


def rounded(x: torch.Tensor, dtype=torch.float64) -> torch.Tensor:
    return values(*quantised(x), x.shape[-1], dtype)


class Fp4Case(Int8Case):
    """Sequences of ``lens`` keys in one paged 4-bit cache; rows that no sequence owns hold the largest codes, block scales of
    no number and the exponent of no number, so that whatever reads one of them shows.  ``exponents``: (n, hkv, generator) ->
    the values' exponent bytes [n, hkv]."""

    def __init__(self, lens, hkv, d, page_size, seed=0, device="cuda", extra_pages=3, exponents=None, first_page=1):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hkv, self.d, self.page_size, self.device = list(lens), hkv, d, page_size, device
        per = [-(-n // page_size) for n in lens]
        total = sum(per) + extra_pages + first_page
        order = (torch.randperm(total - first_page, generator=g) + first_page).tolist()
        self.data = torch.full((total, 2, hkv, page_size, d // 2), 0x77, dtype=torch.uint8, device=device)
        self.scales = torch.full((total, 2, hkv, page_size, d // 16), 0x7f, dtype=torch.uint8, device=device)
        self.exponents = torch.full((total, 2, hkv, page_size), 255, dtype=torch.uint8, device=device)
        self.tables = []
        for n, count in zip(lens, per):
            pages = [order.pop() for _ in range(count)]
            self.tables.append(pages)
            if n == 0:
                continue
            at = torch.arange(n)
            codes = torch.randint(0, 256, (n, 2, hkv, d // 2), generator=g).to(torch.uint8)
            # scales from 1 to 15: a key's dot product with a normal query is some 30 times the head's root
            scales = torch.randint(0x38, 0x58, (n, 2, hkv, d // 16), generator=g).to(torch.uint8)
            units = torch.randint(120, 124, (n, 2, hkv), generator=g).to(torch.uint8)
            if exponents is not None:
                units[:, 1] = exponents(n, hkv, g)
            page, row = torch.tensor(pages)[at // page_size].to(device), (at % page_size).to(device)
            self.data[page, :, :, row] = codes.to(device)
            self.scales[page, :, :, row] = scales.to(device)
            self.exponents[page, :, :, row] = units.to(device)

    def cache(self):
        return ops.Fp4Cache(self.data, self.scales.view(torch.float8_e4m3fn), self.exponents)

    def alone(self, s):
        """Sequence s by itself."""
        one = Fp4Case.__new__(Fp4Case)
        one.__dict__.update(self.__dict__)
        one.tables, one.lens = [self.tables[s]], [self.lens[s]]
        return one

    def rows(self, s, n):
        """(keys, values) [n, Hkv, D] of sequence s in 64 bits."""
        at = torch.arange(n, device=self.device)
        page = torch.tensor(self.tables[s] or [0], device=self.device)[at // self.page_size]
        row = at % self.page_size
        x = values(self.data[page, :, :, row], self.scales.view(torch.float8_e4m3fn)[page, :, :, row],
                   self.exponents[page, :, :, row], self.d)
        return x[:, 0], x[:, 1]
