"""A paged cache with sequences of given rows and lengths on the GPU, the library's calls on it, and the same in 64 bits."""
import torch

from mm_amx_b200 import capi

BF16 = 2.0 ** -8        # half a step of bf16, relative


class Paged:
    """rows, lens: of each sequence.  layout: how the pool lies ("heads": [page, head, place], "places": [page, place, head], "padded": gaps everywhere).
    What no token of a sequence fills is NaN (bf16) or any byte under the factor NaN (int8), and page numbers behind a sequence are wild."""

    def __init__(self, rows, lens, Hkv=2, G=2, D=64, page=16, int8=False, layout="heads", seed=0, extra=0, row0=0, one_row=False, std=1.0):
        self.rows, self.lens, self.Hkv, self.G, self.D, self.P, self.int8 = list(rows), list(lens), Hkv, G, D, page, int8
        self.H, self.B = Hkv * G, len(rows)
        g = self.g = torch.Generator(device="cuda")
        g.manual_seed(seed + 1000 * sum(lens) + D + page)
        need = [-(-n // page) for n in lens]
        self.pages, width = sum(need) + 2, max(need + [1]) + 1
        es = 1 if int8 else 2
        dt = torch.int8 if int8 else torch.bfloat16
        pad = 16 // es if layout == "padded" else 0
        shape = (self.pages, page, Hkv) if layout == "places" else (self.pages, Hkv, page)
        self.raw = [torch.empty(shape[0], shape[1] + (1 if pad else 0), shape[2], D + pad, dtype=dt, device="cuda") for _ in range(2)]
        views = [t[:, :shape[1], :, :D] for t in self.raw]
        self.pool = [t.transpose(1, 2) if layout == "places" else t for t in views]          # [page, head, place, D]
        order = torch.randperm(self.pages, generator=g, device="cuda").tolist()
        self.ids = [order[sum(need[:b]):sum(need[:b + 1])] for b in range(self.B)]
        table = torch.tensor([2 ** 31 - 1, -1, -2 ** 31, self.pages], dtype=torch.int32, device="cuda").repeat(self.B, width)[:, :width + 3].contiguous()
        for b, ids in enumerate(self.ids):
            table[b, :len(ids)] = torch.tensor(ids, dtype=torch.int32, device="cuda")
        self.table = table
        # the scales of all pages, with a gap between pages
        self.scales = [torch.full((self.pages, Hkv + 1), float("nan"), device="cuda") for _ in range(2)] if int8 else None
        for i in range(2):
            if int8:
                self.raw[i].random_(-128, 128, generator=g)
            else:
                self.raw[i].fill_(float("nan"))
            for b, n in enumerate(lens):
                for j, pg in enumerate(self.ids[b]):
                    k = min(page, n - j * page)
                    x = torch.randn(Hkv, k, D, generator=g, device="cuda") * std
                    if int8:
                        s = x.abs().amax((1, 2)) / 127
                        self.scales[i][pg, :Hkv] = s
                        self.pool[i][pg, :, :k] = (x / s[:, None, None]).round().clamp(-127, 127).to(torch.int8)
                    else:
                        self.pool[i][pg, :, :k] = x.to(torch.bfloat16)
        starts = [row0]
        for r in rows:
            starts.append(starts[-1] + r)
        self.starts, self.T = starts, starts[-1] + extra
        self.row_start = None if one_row else torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        # q as the first heads of a wider row
        self.wide = torch.randn(self.T, self.H + 2 * Hkv, D, generator=g, device="cuda").to(torch.bfloat16)
        self.q = self.wide[:, :self.H]
        self.out = torch.full((self.T, self.H + 1, D), 7.0, dtype=torch.bfloat16, device="cuda")

    def cache(self, **kw):
        k, v = self.pool
        es = k.element_size()
        c = dict(pages=self.pages, page_tokens=self.P, Hkv=self.Hkv, D=self.D, dtype=capi.S8 if self.int8 else capi.BF16, k=k.data_ptr(), v=v.data_ptr(),
                 page_stride=k.stride(0) * es, head_stride=k.stride(1) * es, token_stride=k.stride(2) * es, B=self.B, max_pages=self.table.shape[1],
                 page_table=self.table.data_ptr(), table_stride=self.table.stride(0) * 4, seq_lens=self.seq_lens.data_ptr())
        if self.int8:
            c.update(k_scale=self.scales[0].data_ptr(), v_scale=self.scales[1].data_ptr(), scale_page_stride=self.scales[0].stride(0) * 4)
        c.update(kw)
        return capi.PagedCache(**c)

    def attend(self, scale=None, window=0, sinks=0, stream=None, max_rows=None, out=None, cache=None):
        out = self.out if out is None else out
        c = self.cache() if cache is None else cache
        a = capi.PagedAttention(cache=capi.pointer(c), T=self.T, max_rows=max(self.rows) if max_rows is None else max_rows, H=self.H,
                                row_start=None if self.row_start is None else self.row_start.data_ptr(), q=self.q.data_ptr(),
                                q_row_stride=self.q.stride(0) * 2, q_head_stride=self.q.stride(1) * 2, out=out.data_ptr(),
                                out_row_stride=out.stride(0) * 2, out_head_stride=out.stride(1) * 2,
                                scale=self.D ** -0.5 if scale is None else scale, window=window, sinks=sinks)
        capi.paged_attention(a, stream=stream)
        return out[:, :self.H]

    def cached(self, i, b):
        """k (i = 0) or v of sequence b as it stands in the cache: [head, token, D] in 64 bits"""
        if not self.ids[b]:
            return torch.zeros(self.Hkv, 0, self.D, dtype=torch.float64, device="cuda")
        x = self.pool[i][self.ids[b]].double()
        if self.int8:
            x = x * self.scales[i][self.ids[b], :self.Hkv].double()[..., None, None]
        return x.transpose(0, 1).reshape(self.Hkv, -1, self.D)[:, :self.lens[b]]

    def attended(self, scale=None, window=0, sinks=0):
        """(result, sum of p |v| / sum of p) of each owned row, in 64 bits; masked tokens take no part, whatever they hold"""
        scale = self.D ** -0.5 if scale is None else scale
        ref = torch.full((self.T, self.H, self.D), 7.0, dtype=torch.float64, device="cuda")
        mag = torch.zeros_like(ref)
        for b in range(self.B):
            r, n = self.rows[b], self.lens[b]
            if not r:
                continue
            k, v = self.cached(0, b), self.cached(1, b)
            q = self.q[self.starts[b]:self.starts[b] + r].double().reshape(r, self.Hkv, self.G, self.D)
            place = torch.arange(n - r, n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None]
            seen = j <= place
            if window:
                seen &= (j > place - window) | (j < sinks)
            s = torch.einsum("rhgd,hjd->rhgj", q, k) * scale
            s = torch.where(seen[:, None, None], s, float("-inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)) if n else s
            p = torch.where(seen[:, None, None], p, 0)
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, 1, total)
            rows = slice(self.starts[b], self.starts[b] + r)
            bad = ~torch.isfinite(v)
            fine = torch.where(bad, 0, v)
            ref[rows] = torch.einsum("rhgj,hjd->rhgd", p, fine).reshape(r, self.H, self.D)
            mag[rows] = torch.einsum("rhgj,hjd->rhgd", p, fine.abs()).reshape(r, self.H, self.D)
            if bad.any():            # a value that is no number reaches the rows that see it
                hit = torch.einsum("rhgj,hjd->rhgd", (p > 0).double(), bad.double()) > 0
                ref[rows] = torch.where(hit.reshape(r, self.H, self.D), float("nan"), ref[rows])
        return ref, mag

    def check(self, got, ref, mag):
        """p is rounded to bf16 (half a step each), the result once more; exp and the fp32 scores are off by 3e-4 at most"""
        got = got.double()
        assert torch.equal(torch.isfinite(got), torch.isfinite(ref)), "rows that are no numbers differ"
        fine = torch.isfinite(ref)
        over = ((got - ref).abs() - (BF16 * (mag + ref.abs()) * (1 + 2 ** -7) + 3e-4 * mag))[fine]
        assert over.numel() == 0 or float(over.max()) <= 0, "off by %.3g more than allowed" % float(over.max())
        for r in range(self.T):          # rows of no sequence keep what they held
            if r < self.starts[0] or r >= self.starts[-1]:
                assert bool((got[r] == 7.0).all())
        assert bool((self.out[:, self.H:] == 7.0).all())
