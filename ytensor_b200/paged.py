"""Keys and values of many sequences in pages: the cache of a program that serves requests of different lengths, drafts
tokens ahead, or searches with beams.

A pool holds the keys and values of all layers, [layers, pages, kv_heads, page, dim]. A slot is one sequence: position p lies
in row p % page of the page that table[slot, p // page] names; the slot holds the first held[slot] entries of its row of the
table, and lens[slot] positions are written. refs[page] counts the slots that hold a page: a fork shares pages instead of
copying them, and `reserve` replaces those that would be written while others hold them too. YTensor has one contiguous
cache per model (reference example/qwen3/src/qwen3.cpp:70-126) and no counterpart.

Everything lives on the device and no call waits for it, so that a step can be captured in a CUDA graph and replayed at any
lengths. A step that drafts tokens:

    cache.reserve(counts)                                    # once, for all layers
    for layer ...: o = cache.attend(layer, q, starts, k, v, parents=parents)
    cache.keep(kept, accepted)                               # once, for all layers

What only the device can see to be wrong (no free page, an index out of its range, a write into a shared page) is left out
and noted in `status`; `check()` reads it. Calls on one cache follow one another (one stream, or events between streams).
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib
from ._lib import check, lib
from .api import _dt, _require_cuda

_FOUR, _EIGHT = struct.Struct("4q").pack, struct.Struct("8q").pack
FULL, INVALID, SHARED = 1, 2, 4  # bits of `status`
_TEXT = {FULL: "too few free pages: nothing was reserved or compacted",
         INVALID: "an index out of its range, a position without a page, or a tree that is none",
         SHARED: "rows for a page that other slots hold too (reserve comes first)"}


class _Pages(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_strides", C.c_int64 * 4), ("v_strides", C.c_int64 * 4),
                *((n, C.c_void_p) for n in ("table", "lens", "held", "refs", "status", "scratch")),
                *((n, C.c_int) for n in ("layers", "pages", "page", "kv_heads", "dim", "slots", "max_pages", "dtype"))]


def _bad(text: str):
    return _lib.YtCudaInvalidArgument(_lib.INVALID_ARG, text)


class PagedCache:
    def __init__(self, layers: int, pages: int, page: int, kv_heads: int, dim: int, slots: int, max_pages: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        """An empty cache: `pages` pages of `page` positions, `slots` sequences of at most max_pages pages each."""
        shape = (layers, pages, kv_heads, page, dim)
        self._set(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                  *(torch.zeros(s, dtype=torch.int32, device=device) for s in ((slots, max_pages), slots, slots, pages)))

    @classmethod
    def over(cls, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, held: torch.Tensor,
             refs: torch.Tensor) -> "PagedCache":
        """A cache over tensors that are there already. k and v may have any strides (a pool laid out
        [layers, pages, page, kv_heads, dim] is handed in transposed) but a unit stride along dim."""
        self = cls.__new__(cls)
        self._set(k, v, table, lens, held, refs)
        return self

    def _set(self, k, v, table, lens, held, refs):
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype:
            raise _bad("paged cache: k and v are [layers, pages, kv_heads, page, dim] of one shape and type")
        if 0 in (k.shape[0], *k.shape[2:]):
            raise _bad(f"paged cache: an empty axis in {list(k.shape)}")
        for t in (k, v):
            if t.shape[-1] > 1 and t.stride(-1) != 1:
                raise _bad("paged cache: k and v need a unit stride along dim")
        slots = lens.numel()
        for name, t, shape in (("table", table, (slots, table.shape[-1] if table.dim() else 0)), ("lens", lens, (slots,)),
                               ("held", held, (slots,)), ("refs", refs, (k.shape[1],))):
            if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
                raise _bad(f"paged cache: {name} is a contiguous int32 tensor {list(shape)}")
        if len({t.device for t in (k, v, table, lens, held, refs)}) != 1:
            raise _bad("paged cache: tensors on different devices")
        _require_cuda(k)
        self.k, self.v, self.table, self.lens, self.held, self.refs = k, v, table, lens, held, refs
        self.layers, self.pages, self.kv_heads, self.page, self.dim = k.shape
        self.slots, self.max_pages, self.dtype, self.device = slots, table.shape[1], k.dtype, k.device
        self._index, self._per_slot, self._bounds, self._lib = k.get_device(), (slots,), (slots + 1,), lib()
        self._space = None, 0  # (rows, heads) of the last attend() and the bytes it works in
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        c = _Pages(k.data_ptr(), v.data_ptr(), tuple(k.stride()[:4]), tuple(v.stride()[:4]), table.data_ptr(), lens.data_ptr(),
                   held.data_ptr(), refs.data_ptr(), self.status.data_ptr(), None, self.layers, self.pages, self.page,
                   self.kv_heads, self.dim, self.slots, self.max_pages, _dt(k))
        self._scratch = torch.zeros(max(4, self._lib.ytcuda_pages_scratch(C.addressof(c)) // 4), dtype=torch.int32, device=k.device)
        c.scratch = self._scratch.data_ptr()
        self._c, self._at = c, C.addressof(c)

    # ------------------------------------------------------------------ checks of arguments
    # (What they cost is most of what a small call costs: each attribute is asked for once, and one comparison says that all is well.)
    def _stream(self) -> int:
        device = torch._C._cuda_getDevice()
        if device != self._index:
            raise _bad(f"paged cache: it lies on {self.device}, which is not the current device")
        return torch._C._cuda_getCurrentRawStream(device)

    def _ints(self, t, name: str, shape: tuple) -> int:
        if t.dtype is not torch.int32 or t.shape != shape or t.get_device() != self._index or not t.is_contiguous():
            raise _bad(f"paged cache: {name} is a contiguous int32 tensor {list(shape)} on {self.device}")
        return t.data_ptr()

    def _rows(self, t, name: str, shape: tuple) -> tuple:
        """Strides."""
        st = t.stride()
        if t.shape != shape or t.dtype is not self.dtype or t.get_device() != self._index or (st[2] != 1 and shape[2] > 1):
            raise _bad(f"paged cache: {name} is {self.dtype} {list(shape)} with a unit stride along dim, on {self.device}; "
                       f"got {t.dtype} {list(t.shape)}, strides {list(st)}, on {t.device}")
        return st

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.layers:
            raise _bad(f"paged cache: layer {layer} of {self.layers}")
        return layer

    # ------------------------------------------------------------------ pages
    def reserve(self, counts: torch.Tensor) -> None:
        """Room for counts[slot] more positions behind lens[slot] (int32 [slots]; 0: the slot stays as it is). Free pages are
        handed out in ascending order, slot by slot, for new entries of the table and for those that the new positions go to and
        other slots hold too; of the page that the next position falls inside the slot's rows are copied. (b slots that share a
        page and ask in one call get b pages.) All slots get their pages or, with FULL in `status`, none."""
        check(self._lib.ytcuda_pages_reserve(self._at, self._ints(counts, "counts", self._per_slot), self._stream()))

    def fork(self, source: torch.Tensor) -> None:
        """All slots at once: slot s becomes a copy of slot source[s] as it was before (int32 [slots]; its own number: it stays
        as it is, -1: it is emptied). The copy holds the same pages up to its length; nothing is moved."""
        check(self._lib.ytcuda_pages_fork(self._at, self._ints(source, "source", self._per_slot), None, self._stream()))

    def free(self, gone: torch.Tensor) -> None:
        """Empties the slots with gone[slot] != 0 (int32 [slots]); pages that nobody else holds are free again."""
        check(self._lib.ytcuda_pages_fork(self._at, None, self._ints(gone, "gone", self._per_slot), self._stream()))

    def keep(self, kept: torch.Tensor, accepted: torch.Tensor | None = None, *, base: torch.Tensor | None = None) -> None:
        """Of the rows behind position base[slot] (int32 [slots], default lens) the first kept[slot] of accepted [slots, depth]
        stay, in every layer: row base + accepted[slot, j] moves to base + j, and lens becomes base + kept. Numbers of
        accepted rows ascend along a row; without `accepted` the first kept[slot] rows stay where they are. The pages behind
        stay with the slot, for the next drafted rows."""
        depth = accepted.shape[-1] if accepted is not None and accepted.dim() else 0
        kept_at = self._ints(kept, "kept", self._per_slot)
        check(self._lib.ytcuda_pages_keep(
            self._at, kept_at,  # (no columns: nothing of it is read, but it is not "without accepted")
            None if accepted is None else self._ints(accepted, "accepted", (self.slots, depth)) or kept_at, depth,
            None if base is None else self._ints(base, "base", self._per_slot), self._stream()))

    def compact(self, into: "PagedCache") -> None:
        """The pages in use, in ascending order, become pages 0, 1, .. of another (smaller, larger, differently laid out) cache of
        the same slots, and its table, lens, held and refs those of this one. FULL in its `status`: its pool is too small,
        nothing was written. The two may be views of one pool without an element in common."""
        if into._index != self._index:
            raise _bad("paged cache: compact into a cache on another device")
        check(self._lib.ytcuda_pages_compact(self._at, into._at, self._stream()))

    # ------------------------------------------------------------------ one layer
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor) -> None:
        """Stores rows of new tokens: row starts[s] + i of k and v [rows, kv_heads, dim] goes to position lens[s] + i of slot s
        (starts int32 [slots + 1]). lens stays until `keep`, so that every layer of a step writes the same places."""
        rows = k.shape[0] if k.dim() else 0
        shape = (rows, self.kv_heads, self.dim)
        kr, kh, _ = self._rows(k, "k", shape)
        vr, vh, _ = self._rows(v, "v", shape)
        check(self._lib.ytcuda_pages_append(self._at, self._layer(layer), k.data_ptr(), v.data_ptr(), _FOUR(kr, kh, vr, vh),
                                            self._ints(starts, "starts", self._bounds), rows, self._stream()))

    def attend(self, layer: int, q: torch.Tensor, starts: torch.Tensor, k: torch.Tensor | None = None,
               v: torch.Tensor | None = None, *, parents: torch.Tensor | None = None, scale: float = 0.0,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of new rows: q [rows, heads, dim], rows starts[s] .. starts[s + 1] - 1 are the nodes of slot s, node i at
        position lens[s] + i. A node sees the lens[s] positions of its sequence, itself and its ancestors: parents (int32
        [rows]) names for each row a smaller node of its slot, or -1 where it follows the sequence itself; at most 1024 nodes
        a slot. Without parents the nodes are a chain (the next token, or a piece of a prompt), of any length. heads is a
        multiple of kv_heads; dim is at most 256. k and v [rows, kv_heads, dim] are stored behind the sequences as by
        `append`, in the same call; without them they are in the pages already. scale 0: 1 / sqrt(dim).

        Scores, softmax and sums are fp32; in the 16-bit types the weights are rounded to the type where they meet the values
        (half a step of each: 2^-8 in bf16, 2^-11 in fp16, where one below 2^-32 of a row's largest may count as zero and take
        an infinity along as NaN). Results are rounded to nearest even. A call whose rows, over full rows of the table, are
        more work than it can count is refused (include/ytcuda.h says from where on). Rows behind starts[slots] are not
        written. What a node does not see may be infinite or no number; in fp32 a node that sees an infinity, or a number
        within 2^-12 of the largest, may get NaN. `out` has no element in common with q, k or v, and its rows and heads none
        with one another."""
        stream = self._stream()
        if q.dim() != 3 or q.shape[1] % self.kv_heads:
            raise _bad(f"paged cache: q is [rows, heads, dim] with heads a multiple of {self.kv_heads}, got {list(q.shape)}")
        rows, heads, dim = shape = q.shape
        if dim != self.dim:
            raise _bad(f"paged cache: q has dim {dim}, the cache {self.dim}")
        qr, qh, _ = self._rows(q, "q", shape)
        if out is None:
            out = torch.empty_like(q)
            if out.stride(2) != 1:  # (rows of q that overlap)
                out = torch.empty(shape, dtype=q.dtype, device=q.device)
            o_row, o_head, _ = out.stride()
        else:
            o_row, o_head, _ = self._rows(out, "out", shape)
        if k is not None and v is not None:
            new = (rows, self.kv_heads, dim)
            kr, kh, _ = self._rows(k, "k", new)
            vr, vh, _ = self._rows(v, "v", new)
            kp, vp, strides = k.data_ptr(), v.data_ptr(), _EIGHT(qr, qh, o_row, o_head, kr, kh, vr, vh)
        elif k is None and v is None:
            kp, vp, strides = None, None, _EIGHT(qr, qh, o_row, o_head, 0, 0, 0, 0)
        else:
            raise _bad("paged cache: k and v come together")
        known = self._space
        if known[0] != (rows, heads):
            known = self._space = (rows, heads), self._lib.ytcuda_pages_attend_workspace(self._at, rows, heads)
        size = known[1]
        # (its own for every call: two streams, or two captured graphs, never share it)
        space = self.status.new_empty((size + 3) // 4)
        check(self._lib.ytcuda_pages_attend(self._at, self._layer(layer), q.data_ptr(), out.data_ptr(), kp, vp, strides,
                                            self._ints(starts, "starts", self._bounds),
                                            None if parents is None else self._ints(parents, "parents", (rows,)), rows, heads,
                                            scale, space.data_ptr(), size, stream))
        return out

    def check(self) -> None:
        """Raises what the device has noted since the last check (waits for the current stream): what `status` says of this cache,
        and a wait of a kernel on this device that ran out (YtCudaError with status TIMEOUT: rows of an attend() may be
        unwritten)."""
        with torch.cuda.device(self._index):
            waits = self._lib.ytcuda_device_status(torch.cuda.current_stream().cuda_stream)
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
        said = [t for b, t in _TEXT.items() if bits & b]
        if waits != _lib.OK:
            raise _lib.YtCudaError(waits, "paged cache: " + "; ".join([_lib.last_error() or "a wait on the device ran out", *said]))
        if said:
            raise _lib.YtCudaError(_lib.INVALID_ARG, "paged cache: " + "; ".join(said))
