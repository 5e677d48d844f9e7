"""Example banks: predictions from all example windows rather than the few hundred that an exact GP can hold.

The reference's AGPR draws N = 5000 candidate windows and trains on a tenth of them (agpr.py:92-146).  An ExampleBank keeps every
one, in 4 or 8 bits, and answers a window with the kernel-weighted mean of what belongs to those like it: the same sum as
gpsr_predict's, normalised over the examples, which is what makes a solve unnecessary.  Everything runs in the bank_* functions
of ops (gpsr_bank_* of include/gpsr.h); this class keeps the pages.
"""
import torch

from . import _lib, ops


class ExampleBank:
    """rows: how many examples it can hold (more are refused); dim: columns of a key and of a value (padded to what the kernels
    take); kernel_id: ops.RBF or ops.LINEAR."""

    def __init__(self, rows, dim, heads=1, page_rows=64, bits=4, kernel_id=ops.RBF, device=None):
        wide = [d for d in ops.BANK_DIMS if d >= dim]
        if not wide or rows < 1:
            raise _lib.GpsrError(f"ExampleBank: {rows} rows of {dim} columns (at most {ops.BANK_DIMS[-1]})")
        self.dim, self.heads, self.capacity, self.page_rows = dim, heads, rows, page_rows
        pages = -(-rows // page_rows)
        self.bank = ops.bank_alloc(pages, heads, wide[0], page_rows, bits, kernel_id, device)
        dev = self.bank.offset.device
        self.table = torch.arange(pages, dtype=torch.int32, device=dev)[None]
        self.length = torch.zeros(1, dtype=torch.int32, device=dev)
        self.rows = 0

    def _one(self, value):
        return torch.tensor([value], dtype=torch.int32, device=self.length.device)

    def _rows(self, x):
        """[n,dim] or [n,heads,dim] -> [1,n,heads,padded dim]."""
        if x.dim() == 2:
            x = x[:, None]
        if x.dim() != 3 or x.shape[1:] != (self.heads, self.dim):
            raise _lib.GpsrError(f"ExampleBank: expected [n,{self.heads},{self.dim}] rows, got {tuple(x.shape)}")
        pad = self.bank.centroid.shape[-1] - self.dim
        return (torch.nn.functional.pad(x, (0, pad)) if pad else x)[None]

    def append(self, keys, values):
        """Rounds and stores [n,dim] (or [n,heads,dim]) keys and values behind the rows that are there."""
        n = keys.shape[0]
        if self.rows + n > self.capacity:
            raise _lib.GpsrError(f"ExampleBank: {self.rows} + {n} rows are more than the {self.capacity} it was made for")
        ops.bank_write(self.bank, self.table, self._one(self.rows), self._one(n), self._rows(keys), self._rows(values))
        self.rows += n
        self.length.fill_(self.rows)
        return self

    def read(self, start, count, dtype=torch.float32):
        """The keys and values that rows start .. start + count - 1 hold, [count,heads,dim] each; zeros behind the last row."""
        if start < 0:
            raise _lib.GpsrError(f"ExampleBank: rows are counted from 0, got {start}")
        k, v = ops.bank_read(self.bank, self.table, self._one(start), self._one(min(count, self.rows - start)), count, dtype)
        return k[0, ..., :self.dim], v[0, ..., :self.dim]

    def predict(self, queries, scale, pages=None, skip=None, want_lse=False):
        """queries [n,dim] (or [n,heads,dim], or already padded [1,n,q_heads,padded dim]) -> the weighted mean of the values, laid out
        the same.  pages: look at that many pages for each query, the ones whose mean keys suit it best, instead of the whole bank.
        skip [n,2] int32: rows that a query does not see."""
        padded = queries.dim() == 4
        q = queries if padded else self._rows(queries)
        sk = None if skip is None else skip[None].contiguous()
        if pages is None or pages * self.page_rows >= self.rows:
            got = ops.bank_attend(self.bank, self.table, self.length, q, scale, skip=sk, want_lse=want_lse)
        else:
            sel = ops.bank_select(self.bank, self.table, self.length, q, pages, skip=sk)
            got = ops.bank_attend_pages(self.bank, self.table, self.length, q, sel, scale, skip=sk, want_lse=want_lse)
        out, lse = got if want_lse else (got, None)
        if not padded:
            out = out[0, ..., :self.dim] if queries.dim() == 3 else out[0, :, 0, :self.dim]
        return (out, lse[0]) if want_lse else out

    def choose_scale(self, scales, sample=4096, pages=None):
        """The scale of `scales` whose predictions of the bank's own values are best when a row, and what lies within a page of it,
        is left out (mean squared error over `sample` rows spread over the bank; what is not a number is passed over, and refused if
        nothing else is there)."""
        at = torch.arange(0, self.rows, max(1, self.rows // sample), device=self.length.device)
        keys, values = (x[at] for x in self.read(0, self.rows))
        skip = torch.stack([at - self.page_rows, at + self.page_rows + 1], -1).to(torch.int32)
        errors = [float((self.predict(keys, s, pages, skip) - values).square().nanmean()) for s in scales]
        if any(e != e for e in errors):
            raise _lib.GpsrError(f"ExampleBank: none of its {self.rows} rows has a prediction and a value that are numbers")
        return scales[min(range(len(errors)), key=errors.__getitem__)]
