"""Builders and plain 64-bit forms shared by the tests of the paged cache,
shared-prefix attention and sampling."""
from __future__ import annotations

import numpy as np
import torch

import grande_amd as g

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ELEM = {"f32": g.ELEM_F32, "f16": g.ELEM_F16, "bf16": g.ELEM_BF16}


def half_step(dtype) -> float:
    """Half a rounding step of the type, relative to the value."""
    return torch.finfo(dtype).eps / 2


class Pool:
    """A page pool on the GPU filled with noise, with the tables of `lens`
    own rows per sequence and a prefix of `prefix` rows, pages shuffled."""

    def __init__(self, rng, lens, prefix, kv_heads, hd, page, dtype, spare=2, page_pad=0):
        lens = np.asarray(lens)
        own = -(-np.maximum(lens, 0) // page)
        pre = -(-prefix // page)
        total = int(own.sum()) + pre + spare
        ids = rng.permutation(total)
        most = max(1, int(own.max()))
        table = np.zeros((len(lens), most + 1), np.int32)
        at = pre
        for s, n in enumerate(own):
            table[s, :n] = ids[at:at + n]
            at += n
        self.kv_heads, self.hd, self.page, self.dtype = kv_heads, hd, page, dtype
        self.npages, self.max_pages, self.prefix = total, most, prefix
        self.prefix_ids = ids[:pre].astype(np.int32)
        self.table_host, self.lens_host = table, lens.astype(np.int32)
        self.stride = kv_heads * page * hd + page_pad
        gen = torch.Generator().manual_seed(int(rng.integers(1 << 30)))
        self.k_raw, self.v_raw = (torch.randn(total, self.stride, generator=gen).to(TYPES[dtype]).cuda()
                                  for _ in range(2))
        self.table = torch.from_numpy(table).cuda()
        self.lens = torch.from_numpy(self.lens_host).cuda()
        self.prefix_table = torch.from_numpy(np.ascontiguousarray(self.prefix_ids if pre else [0], np.int32)).cuda()

    def view(self, raw):
        n = self.kv_heads * self.page * self.hd
        return raw[:, :n].view(self.npages, self.kv_heads, self.page, self.hd)

    @property
    def k(self):
        return self.view(self.k_raw)

    @property
    def v(self):
        return self.view(self.v_raw)

    def kv(self) -> g.PagedKv:
        return g.PagedKv(self.k_raw.data_ptr(), self.v_raw.data_ptr(), self.npages, self.kv_heads, self.page, self.hd,
                         ELEM[self.dtype], self.stride)

    def batch(self, tokens, start=None, **over) -> g.PagedBatch:
        a = dict(nseq=len(self.lens_host), tokens=tokens, lens_ptr=self.lens.data_ptr(),
                 table_ptr=self.table.data_ptr(), max_pages=self.max_pages,
                 start_ptr=start.data_ptr() if start is not None else None,
                 prefix_table_ptr=self.prefix_table.data_ptr(), prefix_len=self.prefix,
                 table_ld=self.table_host.shape[1])
        a.update(over)
        return g.PagedBatch(**a)

    def rows(self, raw, seq):
        """The own rows of a sequence [len][kv_heads][hd] in 64 bits, from the current contents."""
        x = self.view(raw).double().cpu()
        n = int(self.lens_host[seq])
        r = np.arange(n)
        return x[torch.from_numpy(self.table_host[seq, r // self.page].astype(np.int64)), :, torch.from_numpy(r % self.page)]

    def prefix_rows(self, raw):
        x = self.view(raw).double().cpu()
        r = np.arange(self.prefix)
        return x[torch.from_numpy(self.prefix_ids[r // self.page].astype(np.int64)) if self.prefix else [], :,
                 torch.from_numpy(r % self.page)]


def starts(new) -> torch.Tensor:
    return torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()


def rope_table(rows: int, dims: int, theta: float = 1e4) -> torch.Tensor:
    f = theta ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * f
    return torch.stack([ang.cos(), ang.sin()], -1).float()


def plain_rope(x, cs, layout):
    """x [..., hd] float64 by cs [dims / 2][2], pair by pair."""
    y = x.clone()
    hd, n = x.shape[-1], cs.shape[0]
    for i in range(n):
        a, b = {g.ROPE_HALF: (i, i + n), g.ROPE_INTERLEAVED: (2 * i, 2 * i + 1),
                g.ROPE_HEAD_HALF: (i, i + hd // 2)}[layout]
        c, s = float(cs[i, 0]), float(cs[i, 1])
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def plain_norm(x, w, eps):
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return y if w is None else y * w.double().cpu()
