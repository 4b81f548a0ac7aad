"""Ragged-batch cases over a paged cache for the attention tests: pools that hold NaN wherever no row may look, and
the definition in 64 bits with the bound that the kernel's roundings leave."""
from __future__ import annotations

import torch

BAD_PAGE = 0x7FFFFFF0  # table entries that must not be read


class ChunkCase:
    """Sequences with q_lens[b] new tokens as the last of kv_lens[b] cached rows; hidden pages (wholly behind the window
    of every row) hold no page id, rows that nobody sees hold NaN."""

    def __init__(self, *, hq, hkv, d, page, q_lens, kv_lens, window=0, sinks=0, seed=1, spread=1.0):
        self.hq, self.hkv, self.d, self.page, self.window, self.sinks = hq, hkv, d, page, window, sinks
        self.q_lens, self.kv_lens = list(q_lens), list(kv_lens)
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-n // page) for n in kv_lens]
        self.n_pages = sum(need) + 3
        order = torch.randperm(self.n_pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(kv_lens), max(max(need), 1)), BAD_PAGE, dtype=torch.int32, device="cuda")
        shape = (self.n_pages, hkv, page, d)
        self.k = torch.full(shape, float("nan"), dtype=torch.float16, device="cuda")
        self.v = torch.full(shape, float("nan"), dtype=torch.float16, device="cuda")
        self.tokens = sum(q_lens)
        self.q = torch.randn((max(self.tokens, 1), hq * d), generator=g, device="cuda").mul_(spread).half()
        self.kc, self.vc = [], []
        at = 0
        for b, n in enumerate(kv_lens):
            pages = order[at:at + need[b]]
            at += need[b]
            kc = torch.randn((hkv, n, d), generator=g, device="cuda").half()
            vc = torch.randn((hkv, n, d), generator=g, device="cuda").half()
            seen = self.visible(b).any(0) if q_lens[b] and n else torch.zeros(n, dtype=torch.bool, device="cuda")
            for j in range(need[b]):
                s = slice(j * page, min(n, (j + 1) * page))
                if bool(seen[s].any()):
                    self.table[b, j] = pages[j]
                    rows = seen[s][None, :, None]
                    self.k[pages[j], :, : s.stop - s.start] = torch.where(rows, kc[:, s], float("nan"))
                    self.v[pages[j], :, : s.stop - s.start] = torch.where(rows, vc[:, s], float("nan"))
            self.kc.append(kc)
            self.vc.append(vc)
        self.lens = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")

    def visible(self, b):
        """[q_len, kv_len]: which keys each row of sequence b sees."""
        n, nq = self.kv_lens[b], self.q_lens[b]
        pos = torch.arange(n - nq, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None]
        see = key <= pos
        if self.window:
            see &= (pos - key < self.window) | (key < self.sinks)
        return see

    def expected(self, scale=None):
        """(outputs, bound) in 64 bits, [tokens, hq, d].

        The kernel's roundings: a weight to f16 (2^-11 of it, or 2^-25 where it is subnormal; the largest is at least 1),
        the output to f16 (2^-11 of it, or 2^-25), and f32 sums whose error the 2^-12 of the weighted mean of |v| covers
        (scores of |s| < 30 off by 128 * 2^-24 * 30, sums of n/16 terms)."""
        scale = self.d ** -0.5 if scale is None else scale
        out = torch.zeros((max(self.tokens, 1), self.hq, self.d), dtype=torch.float64, device="cuda")
        tol = torch.full_like(out, 2.0 ** -25)
        t = 0
        for b, nq in enumerate(self.q_lens):
            if nq and self.kv_lens[b]:
                see = self.visible(b)
                rows = see.any(1)
                for h in range(self.hq):
                    k, v = self.kc[b][h // (self.hq // self.hkv)].double(), self.vc[b][h // (self.hq // self.hkv)].double()
                    q = self.q[t:t + nq, h * self.d:(h + 1) * self.d].double()
                    s = (q @ k.T * scale).masked_fill(~see, -float("inf"))
                    w = torch.softmax(s[rows], -1)
                    o, a = w @ v, w @ v.abs()
                    out[t:t + nq, h][rows] = o
                    few = see[rows].sum(1, keepdim=True) * 2.0 ** -25 * float(v.abs().max())
                    tol[t:t + nq, h][rows] = 2.0 ** -25 + 2.0 ** -11 * o.abs() + (2.0 ** -11 + 2.0 ** -12) * a + few
            t += nq
        return out[:self.tokens], tol[:self.tokens]

    def cache(self, mfk):
        return mfk.paged_kv(self.k, self.v, self.table, self.lens, n_kv_heads=self.hkv, page_size=self.page, head_dim=self.d)

    def plan(self, f, **kw):
        return f.chunk_plan(self.q_lens, self.kv_lens, n_heads=self.hq, n_kv_heads=self.hkv, head_dim=self.d, page_size=self.page,
                            window=self.window, sinks=self.sinks, **kw)


def check(out, case, scale=None):
    want, tol = case.expected(scale)
    off = (out.double().view(case.tokens, case.hq, case.d) - want).abs()
    assert bool(torch.isfinite(out).all()), "a value that no row sees reached the output"
    worst = float((off - tol).max()) if off.numel() else -1.0
    assert worst <= 0, f"off by {float(off.max()):.3g}, {worst:.3g} over the bound"
