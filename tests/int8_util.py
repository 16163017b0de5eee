"""Plain implementations in 64 bits of the operators in 8-bit integers, and a paged cache with shuffled pages."""

from __future__ import annotations

import torch

from deterministic_inference_b200.engine.batch import AttentionMeta

FLOOR = 2.0 ** -100


def codes_of(x: torch.Tensor):
    """Codes and scales of the last axis' rows, with the float32 operations that define them."""
    x = x.float()
    a = x.abs().amax(-1)
    bad = ~torch.isfinite(a)
    a = torch.where(bad, torch.ones_like(a), a).clamp(min=FLOOR)
    one = torch.ones_like(a)                     # (a tensor: the quotients are rounded, and so are the products)
    codes = torch.round(x * ((one / a) * 127.0)[..., None])
    codes = torch.where(bad[..., None], torch.zeros_like(codes), codes).to(torch.int8)
    return codes, torch.where(bad, torch.full_like(a, float("nan")), a * (one / (127.0 * one)))


class Int8Case:
    """Sequences of ``lens`` keys in one paged int8 cache; rows that no sequence owns hold the largest codes and the scale
    NaN, so that whatever reads one of them shows."""

    def __init__(self, lens, hkv, d, page_size, seed=0, device="cuda", extra_pages=3, value_scales=None, first_page=1):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hkv, self.d, self.page_size, self.device = list(lens), hkv, d, page_size, device
        per = [-(-n // page_size) for n in lens]
        total = sum(per) + extra_pages + first_page
        order = (torch.randperm(total - first_page, generator=g) + first_page).tolist()
        self.data = torch.full((total, 2, hkv, page_size, d), 127, dtype=torch.int8, device=device)
        self.scales = torch.full((total, 2, hkv, page_size), float("nan"), dtype=torch.float32, device=device)
        self.tables = []
        for n, count in zip(lens, per):
            pages = [order.pop() for _ in range(count)]
            self.tables.append(pages)
            if n == 0:
                continue
            at = torch.arange(n)
            codes = torch.randint(-127, 128, (n, 2, hkv, d), generator=g).to(torch.int8)
            scales = torch.rand(n, 2, hkv, generator=g) / 64 + 1 / 128
            if value_scales is not None:
                scales[:, 1] = value_scales(n, hkv, g)
            page = torch.tensor(pages)[at // page_size].to(device)
            row = (at % page_size).to(device)
            self.data[page, :, :, row] = codes.to(device)
            self.scales[page, :, :, row] = scales.to(device)

    def rows(self, s, n):
        """(keys, values) [n, Hkv, D] of sequence s in 64 bits."""
        at = torch.arange(n, device=self.device)
        page = torch.tensor(self.tables[s] or [0], device=self.device)[at // self.page_size]
        row = at % self.page_size
        x = self.data[page, :, :, row].double() * self.scales[page, :, :, row].double()[..., None]
        return x[:, 0], x[:, 1]

    def meta(self, q_lens, kv_lens=None):
        kv_lens = list(self.lens if kv_lens is None else kv_lens)
        width = max(1, max(len(t) for t in self.tables))
        bt = torch.zeros(len(q_lens), width, dtype=torch.int32)
        for b, t in enumerate(self.tables):
            bt[b, :len(t)] = torch.tensor(t, dtype=torch.int32)
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device=self.device)
        cu = [0]
        for n in q_lens:
            cu.append(cu[-1] + n)
        seq = [b for b, n in enumerate(q_lens) for _ in range(n)]
        pos = [max(0, kv - n + i) for n, kv in zip(q_lens, kv_lens) for i in range(n)]
        nd = 0
        while nd < len(q_lens) and q_lens[nd] == 1:
            nd += 1
        return AttentionMeta(block_table=bt.to(self.device), slot_mapping=ints([0] * len(seq)), token_seq=ints(seq),
                             positions=ints(pos), cu_q_lens=ints(cu), seq_lens=ints(kv_lens), q_lens=list(q_lens),
                             kv_lens=kv_lens, num_decode=nd)

    def attention(self, q, q_lens, scale, window=None, kv_lens=None):
        """In 64 bits: the output [T, Hq, D], and how far one in 32 or 16 bits may be off it, [T, 1, 1] each: the largest
        visible |value| of the token's sequence (times an error of the probabilities), and the largest scale * sum |q||k|
        of a score."""
        kv_lens = list(self.lens if kv_lens is None else kv_lens)
        t, hq, d = q.shape
        group = hq // self.hkv
        out = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device)
        vmax = torch.zeros(t, 1, 1, dtype=torch.float64, device=q.device)
        smax = torch.zeros_like(vmax)
        at = 0
        for s, (n, length) in enumerate(zip(q_lens, kv_lens)):
            if length > 0:
                k, v = self.rows(s, length)
                k, v = (x.repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))      # [Hq, L, D]
                keys = torch.arange(length, device=q.device)
                step = max(1, (1 << 25) // (hq * length))
                for r in range(0, n, step):
                    m = min(step, n - r)
                    qs = q[at + r:at + r + m].double().transpose(0, 1)
                    p = torch.arange(length - n + r, length - n + r + m, device=q.device)[:, None]
                    seen = keys <= p
                    if window:
                        seen &= keys > p - window
                    sc = (qs @ k.transpose(1, 2) * scale).masked_fill(~seen, float("-inf"))
                    w = torch.softmax(sc, -1)
                    w = torch.where(seen.any(-1)[:, None], w, torch.zeros_like(w))
                    out[at + r:at + r + m] = (w @ v).transpose(0, 1)
                    mags = (qs.abs() @ k.abs().transpose(1, 2) * abs(scale)).masked_fill(~seen, 0.0)
                    smax[at + r:at + r + m, 0, 0] = mags.amax((0, 2))
                    vmax[at + r:at + r + m, 0, 0] = (seen[None] * v.abs().amax(-1)[:, None]).amax((0, 2))
            at += n
        return out, vmax, smax
