"""The latent attention of a batch of sequences over a paged cache in 8 bits: LatentCache (append, read,
attend) and LatentBatch, over mk_latent_* (csrc/mk_latent.cu, csrc/mk_latent_attend.cu).

The persistent kernel decodes one sequence over a BF16 cache of its own; this is the cache and the
attention of a batch. A token of the cache is a latent of d_c values, which is the key and the value of
every head, and a rotary key of d_r values that all heads share (the absorbed form of the model's
attention). Codes are E4M3 bytes, and each page has one scale for its latents and one for its rotary
keys: the smallest power of two 2^e with |x| <= 448 2^e for what the page holds, e from -32 to 32. It is
anew where a page's first token is written and grows with later ones otherwise, its earlier codes being
rounded to it.
"""
import ctypes

import torch

from fleet import mk
from fleet.rope import _apart, overlap

DTYPES = {torch.bfloat16: 0, torch.float16: 1}
PAGES = (16, 32, 64, 128)
MOST = 2 ** 31 - 1       # what the library counts sequences, pages, rows and heads with has 32 bits


def _beside(a, b):
    """Whether the rows of two 2-D tensors are side by side in longer rows."""
    ld, at = a.stride(0), (b.data_ptr() - a.data_ptr()) // a.element_size()
    return b.stride(0) == ld and ld > 0 and a.shape[1] <= at % ld <= ld - b.shape[1]


class LatentBatch:
    """The sequences of a call: `table` [B, P] int32, the pages of each; `lens` [B] int32, the tokens of
    each, the ones of this step included; `starts` [B + 1] int32, where the rows of each begin in the
    call's tensors (ascending, or results are undefined; rows from starts[B] on belong to nobody), or None for one row each, row b
    being sequence b's. Row i of the n of a sequence is its token lens - n + i.

    The tensors are held and may change between calls (a captured graph reads what they hold then).
    What they say is the device's: a length below 0 counts as 0, and a token past the P pages or in a page
    outside the cache is none: it is not written, reads as zeros and is seen by nobody. (Where a length is past the
    pages, the rows' tokens still go by it, so that the last rows have none.)"""

    def __init__(self, table, lens, starts=None):
        B = lens.shape[0] if lens.dim() == 1 else -1
        if lens.dtype != torch.int32 or B < 0 or not lens.is_contiguous():
            raise ValueError(f"lens: contiguous int32 [B] expected, got {lens.dtype} {tuple(lens.shape)}")
        if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != B or table.shape[1] < 1 or \
                (table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError(f"table: int32 [{B}, P] with unit stride along P expected, got {table.dtype} {tuple(table.shape)}, strides {table.stride()}")
        if starts is not None and (starts.dtype != torch.int32 or tuple(starts.shape) != (B + 1,) or not starts.is_contiguous()):
            raise ValueError(f"starts: contiguous int32 [{B + 1}] expected, got {starts.dtype} {tuple(starts.shape)}")
        if B > MOST or table.shape[1] > MOST:
            raise ValueError(f"a batch has fewer than 2^31 sequences of fewer than 2^31 pages each, got table {tuple(table.shape)}")
        if any(v is not None and v.device != lens.device for v in (table, starts)):
            raise ValueError("table, lens and starts are on one device")
        self.table, self.lens, self.starts = table, lens, starts
        self.n, self.index = B, lens.get_device()
        self.c = mk.MkLatentBatch(table.data_ptr(), lens.data_ptr(), mk._ptr(starts), table.stride(0), B, table.shape[1])
        self.ptr = ctypes.addressof(self.c)
        self.tensors = table, lens, starts


class LatentCache:
    """A cache of `pages` pages of `page` tokens (16, 32, 64 or 128), d_c and d_r multiples of 8 up to 512 and 64.

    `c_codes` [pages, page, d_c] and `r_codes` [pages, page, d_r] uint8 and `scales` [pages, 2] float32
    are the cache's own memory, zero at first; a program may copy, save and fill them. attend's waits end after
    `wait_timeout_s` each; what a block that gave up had still to write is NaN then, and status() says so."""

    def __init__(self, pages, page, d_c, d_r, device="cuda", wait_timeout_s=2.0):
        if page not in PAGES:
            raise ValueError(f"page {page} is one of {PAGES}")
        if not 8 <= d_c <= 512 or d_c % 8 or not 8 <= d_r <= 64 or d_r % 8:
            raise ValueError(f"d_c from 8 to 512 and d_r from 8 to 64, multiples of 8, expected, got {d_c} and {d_r}")
        if pages < 1 or pages * page >= 2 ** 31:
            raise ValueError(f"from 1 page to 2^31 - 1 tokens expected, got {pages} pages of {page}")
        if not 1e-9 <= wait_timeout_s <= 1e9:
            raise ValueError(f"wait_timeout_s {wait_timeout_s} is from 1e-9 to 1e9")
        self.wait_ns = int(wait_timeout_s * 1e9)
        self.pages, self.page, self.d_c, self.d_r = pages, page, d_c, d_r
        self._c = torch.zeros(pages, page, -(-d_c // 128) * 128, dtype=torch.uint8, device=device)
        self._r = torch.zeros(pages, page, 64, dtype=torch.uint8, device=device)
        self.scales = torch.zeros(pages, 2, dtype=torch.float32, device=device)
        self.error = torch.zeros(1, dtype=torch.int32, device=device)
        self.c_codes, self.r_codes = self._c[..., :d_c], self._r[..., :d_r]
        self.device, self.index = self._c.device, self._c.get_device()
        self.c = mk.MkLatent(self._c.data_ptr(), self._r.data_ptr(), self.scales.data_ptr(), pages, page, d_c, d_r)
        self.ptr, self._error = ctypes.addressof(self.c), self.error.data_ptr()
        self.tensors = self._c, self._r, self.scales, self.error
        self._need = {}            # (sequences, rows, heads) -> workspace bytes

    def status(self, raise_on_error=True):
        """{"error": 0, or 1 if a wait of attend ran out since the last reset()} (waits for the current stream)."""
        st = {"error": int(self.error.item())}
        if st["error"] and raise_on_error:
            raise mk.MkError(mk.MK_EDEVICE, "LatentCache.attend: a wait ran out, its outputs hold NaN", st)
        return st

    def reset(self):
        self.error.zero_()

    def _refuse_batch(self, batch, rows):
        if batch.index != self.index:
            raise ValueError(f"the batch is on {batch.lens.device}, the cache on {self.device}")
        if rows > MOST:
            raise ValueError(f"a call has fewer than 2^31 rows, got {rows}")
        raise ValueError(f"without starts a batch has one row for each of its {batch.n} sequences, got {rows} rows")

    def _refuse(self, t, d, name, dtype=None, T=None):
        raise ValueError(f"{name}: {dtype or 'bfloat16 or float16'} [{'rows' if T is None else T}, {d}] with unit stride along its rows on "
                         f"{self.device} expected, got {t.dtype} {tuple(t.shape)}, strides {t.stride()} on {t.device}")

    def append(self, c_kv, k_pe, batch, stream=None):
        """Write the rows' latents c_kv [rows, d_c] (after their norm) and rotary keys k_pe [rows, d_r] (after
        their turn) into the batch's pages, bfloat16 or float16 with any row strides. What is not finite
        becomes NaN and does not count for a scale; values past 448 2^32 saturate. Rows before a sequence's first
        token (more rows than tokens), past its table or in a page outside the cache are left out, and so
        are rows of no sequence. A page is written by one sequence of a call at most; writing tokens again
        (rejected drafts) is an append with shorter lens."""
        if stream is not None:
            with mk.on_stream(c_kv, stream, k_pe, *batch.tensors, *self.tensors):
                return self.append(c_kv, k_pe, batch)
        call, device, current_stream, context = mk.entry("mk_latent_append")
        index = self.index
        if index < 0 or device() != index:
            return mk.off_device("mk_latent_append", index, context, lambda: self.append(c_kv, k_pe, batch))
        dtype = c_kv.dtype
        if c_kv.dim() != 2 or c_kv.shape[1] != self.d_c or c_kv.stride(1) != 1 or c_kv.get_device() != index or dtype not in DTYPES:
            self._refuse(c_kv, self.d_c, "c_kv")
        rows = c_kv.shape[0]
        if k_pe.dim() != 2 or k_pe.shape[1] != self.d_r or k_pe.shape[0] != rows or k_pe.stride(1) != 1 or k_pe.get_device() != index or \
                k_pe.dtype is not dtype:
            self._refuse(k_pe, self.d_r, "k_pe", dtype, rows)
        if batch.index != index or rows > MOST or (batch.starts is None and rows != batch.n):
            self._refuse_batch(batch, rows)
        rc = call(self.ptr, batch.ptr, c_kv.data_ptr(), c_kv.stride(0), k_pe.data_ptr(), k_pe.stride(0), rows, DTYPES[dtype],
                  current_stream(index))
        if rc:
            mk._check(rc, "mk_latent_append")

    def read(self, batch, rows, dtype=torch.bfloat16, out=None, stream=None):
        """(latents [rows, d_c], rotary keys [rows, d_r]) of the batch's rows, code x scale rounded once
        (exact in bfloat16). A whole sequence is lens rows. Tokens that are in no page of the cache read as zeros;
        rows of no sequence are zeros too, or stay as they were in the pair `out`."""
        if stream is not None:
            with mk.on_stream(self._c, stream, *batch.tensors, *self.tensors, *(out or ())):
                return self.read(batch, rows, dtype, out)
        call, device, current_stream, context = mk.entry("mk_latent_read")
        index = self.index
        if index < 0 or device() != index:
            return mk.off_device("mk_latent_read", index, context, lambda: self.read(batch, rows, dtype, out))
        if dtype not in DTYPES:
            raise TypeError(f"dtype is bfloat16 or float16, not {dtype}")
        if batch.index != index or rows > MOST or (batch.starts is None and rows != batch.n):
            self._refuse_batch(batch, rows)
        d_c, d_r, fill = self.d_c, self.d_r, out is None
        if fill:
            c = torch.empty_strided((rows, d_c), (d_c, 1), dtype=dtype, device=self.device)
            r = torch.empty_strided((rows, d_r), (d_r, 1), dtype=dtype, device=self.device)
            ldc, ldr = d_c, d_r
        else:
            c, r = out
            for t, d, name in ((c, d_c, "out[0]"), (r, d_r, "out[1]")):
                if t.dim() != 2 or t.shape[1] != d or t.shape[0] != rows or t.stride(1) != 1 or t.get_device() != index or t.dtype is not dtype:
                    self._refuse(t, d, name, dtype, rows)
            ldc, ldr = c.stride(0), r.stride(0)
            if rows > 1 and (c.stride(0) < self.d_c or r.stride(0) < self.d_r):
                raise ValueError(f"out: rows overlap (strides {c.stride(0)} and {r.stride(0)})")
            if (overlap(c, r) and not _beside(c, r)) or any(t is not None and overlap(o, t) for o in out for t in (*self.tensors, *batch.tensors)):
                raise ValueError("out: its tensors are apart from one another, the cache and the batch")
        rc = call(self.ptr, batch.ptr, c.data_ptr(), ldc, r.data_ptr(), ldr, rows, DTYPES[dtype], fill,
                  current_stream(index))
        if rc:
            mk._check(rc, "mk_latent_read")
        return c, r

    def workspace_bytes(self, n, rows, heads):
        got = self._need.get((n, rows, heads))
        if got is None:
            if max(n, rows, heads) > MOST:
                raise ValueError(f"sequences, rows and heads are below 2^31, got {n}, {rows} and {heads}")
            need = ctypes.c_int64()
            mk._check(mk.lib().mk_latent_attend_workspace(self.ptr, n, rows, heads, ctypes.byref(need)), "mk_latent_attend_workspace")
            if len(self._need) > 4096:
                self._need.clear()
            got = self._need[(n, rows, heads)] = need.value
        return got

    def attend(self, q, batch, scale, out=None, return_lse=False, stream=None):
        """out [rows, heads, d_c] of q [rows, heads, d_c + d_r] (bfloat16 or float16; the absorbed query, then its
        rotary part): softmax over the tokens up to the row's own of scale x (q . (latent, rotary key)), times the
        latents. With return_lse also the log of the sum of the scores' exponentials [rows, heads] float32.
        A row that sees no token gives zeros and -inf. Rows of no sequence stay as they were in `out`
        (undefined in a new tensor). A NaN in a token stays with the rows that see it, an infinity or a NaN in q
        with its row and head, which it makes NaN. Strides of rows and heads may be any. Runs on `stream` (default:
        the current stream); the workspace comes from torch's allocator for each call."""
        if stream is not None:
            with mk.on_stream(q, stream, out, *batch.tensors, *self.tensors):
                return self.attend(q, batch, scale, out, return_lse)
        call, device, current_stream, context = mk.entry("mk_latent_attend_status")
        index = self.index
        if index < 0 or device() != index:
            return mk.off_device("mk_latent_attend", index, context, lambda: self.attend(q, batch, scale, out, return_lse))
        d_c, dtype = self.d_c, q.dtype
        if q.dim() != 3 or q.shape[2] != d_c + self.d_r or q.stride(2) != 1 or q.get_device() != index or dtype not in DTYPES:
            raise ValueError(f"q: bfloat16 or float16 [rows, heads, {d_c + self.d_r}] with unit stride along its values on {self.device} expected, got "
                             f"{q.dtype} {tuple(q.shape)}, strides {q.stride()} on {q.device}")
        rows, heads, _ = q.shape
        if batch.index != index or rows > MOST or (batch.starts is None and rows != batch.n):
            self._refuse_batch(batch, rows)
        if heads > MOST:
            raise ValueError(f"q: fewer than 2^31 heads expected, got {heads}")
        if out is None:
            ot, oh = heads * d_c, d_c
            out = torch.empty_strided((rows, heads, d_c), (ot, oh, 1), dtype=dtype, device=self.device)
        else:
            shape = (rows, heads, d_c)
            if out.shape != shape or out.dtype != dtype or out.get_device() != index or out.stride(2) != 1:
                raise ValueError(f"out: {dtype} {shape} with unit stride along its values on {self.device} expected, got "
                                 f"{out.dtype} {tuple(out.shape)}, strides {out.stride()} on {out.device}")
            if not _apart(shape, out.stride()):
                raise ValueError(f"out: heads overlap (strides {out.stride()}, {d_c} values)")
            if any(t is not None and overlap(out, t) for t in (q, *self.tensors, *batch.tensors)):
                raise ValueError("out is apart from q, the cache and the batch")
            ot, oh, _ = out.stride()
        lse = torch.empty_strided((rows, heads), (heads, 1), dtype=torch.float32, device=self.device) if return_lse else None
        nbytes = self._need.get((batch.n, rows, heads)) or self.workspace_bytes(batch.n, rows, heads)
        ws = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=self.device)
        qt, qh, _ = q.stride()
        rc = call(self.ptr, batch.ptr, q.data_ptr(), qt, qh, rows, heads, DTYPES[dtype], scale, out.data_ptr(), ot, oh,
                  lse.data_ptr() if return_lse else None, ws.data_ptr(), nbytes, self._error, self.wait_ns, current_stream(index))
        if rc:
            mk._check(rc, "mk_latent_attend_status")
        return (out, lse) if return_lse else out
