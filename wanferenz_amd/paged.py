"""A paged key-value cache: the write of new tokens, the attention that reads it, and the
eviction of what attention has weighed least.

The reference keeps one contiguous row of KV latents per sequence
(wanferenz/model/architecture.py:596-600) and attends to selected rows of it
(``kernels.sparse_attn``); this cache has no counterpart there.  Slot t of sequence b lies in
row t % page_size of page ``table[b, t // page_size]``, so sequences of any length share one
pool.  K and V are separate heads, grouped under the query heads, or one latent row that
serves as both (``v=None``, as sparse_attn's rows do).  An e4m3 cache holds one float32 scale
for each row, by act_quant's rule over the whole row (max(amax, 1e-4) / 448).

A decode loop::

    cache = PagedKV.empty(pages, 64, kv_heads=8, head_dim=128, track=True, device=dev)
    cache.write(k, v, table, lens, position=pos)        # the step's new tokens
    o = cache.attend(q, table, lens + 1, scale, accumulate=True)
    lens = cache.evict(table, lens + 1, keep=4096, first=4, recent=1024)

Every call runs on the current stream of the cache's device, allocates only its outputs, (unless
given) its workspace and copies of tables and lengths that are not contiguous and of rows that are not
16-byte aligned, never synchronises, and can be captured in a graph.  The operators
are for serving: they have no gradients.
"""

from __future__ import annotations

import ctypes

import torch

from . import _native as N

_E4M3 = torch.float8_e4m3fn
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream
_I64x3 = ctypes.c_int64 * 3


class WzPagedKV(ctypes.Structure):
    """wz_paged_kv of include/wanferenz_amd.h."""

    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("weights", ctypes.c_void_p), ("positions", ctypes.c_void_p),
                ("pages", ctypes.c_int64), ("page_size", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("head_dim", ctypes.c_int32), ("dtype", ctypes.c_int32)]


class PagedKV:
    """A cache over the caller's pools (``empty`` allocates them):

    k, v       [pages, kv_heads, page_size, head_dim] bf16 or e4m3; v None: one row is K and V
    k_scale, v_scale   float32 [pages, kv_heads, page_size], e4m3 pools only
    weights    float32, the same shape: the attention weight each slot was given so far
    positions  int32, the same shape: the token position that each slot holds
               (weights and positions together make the cache a tracked one)

    Head dims are 64, 128 and 256, or 128, 256 and 512 with v None; page sizes powers of two
    from 16 to 1024.  Table entries outside [0, pages) are pages that hold nothing.  Tables,
    lengths, starts, counts and positions of the calls are int32 tensors on the pools' device.
    """

    def __init__(self, k, v=None, *, k_scale=None, v_scale=None, weights=None, positions=None):
        if k.dim() != 4:
            raise ValueError(f"PagedKV: k must be [pages, kv_heads, page_size, head_dim], got {list(k.shape)}")
        if k.dtype not in (torch.bfloat16, _E4M3):
            raise TypeError(f"PagedKV: bf16 or float8_e4m3fn pools expected (got {k.dtype})")
        if v is not None and (v.shape != k.shape or v.dtype != k.dtype):
            raise ValueError(f"PagedKV: v {list(v.shape)} {v.dtype} does not match k {list(k.shape)} {k.dtype}")
        quantised = k.dtype == _E4M3
        if (k_scale is not None) != quantised or (v_scale is not None) != (quantised and v is not None):
            raise ValueError("PagedKV: k_scale and v_scale belong to e4m3 pools, one for each of k and v")
        if (weights is None) != (positions is None):
            raise ValueError("PagedKV: a tracked cache has both weights and positions")
        slots = k.shape[:3]
        for name, t, dt in (("k_scale", k_scale, torch.float32), ("v_scale", v_scale, torch.float32),
                            ("weights", weights, torch.float32), ("positions", positions, torch.int32)):
            if t is not None and (t.shape != slots or t.dtype != dt):
                raise ValueError(f"PagedKV: {name} must be {dt} {list(slots)}, got {t.dtype} {list(t.shape)}")
        held = [t for t in (k, v, k_scale, v_scale, weights, positions) if t is not None]
        for t in held:
            if not t.is_cuda:
                raise RuntimeError("wanferenz_amd kernels run on the GPU only (got a CPU tensor); "
                                   "there is no CPU fallback in this package")
            if not t.is_contiguous():
                raise ValueError("PagedKV: the pools must be contiguous")
            if t.device != k.device:
                raise ValueError("PagedKV: the pools are on different devices")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.weights, self.positions = weights, positions
        self.device = k.device
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        d = WzPagedKV(N.ptr(k), N.ptr(v), N.ptr(k_scale), N.ptr(v_scale), N.ptr(weights), N.ptr(positions), self.pages,
                      self.page_size, self.kv_heads, self.head_dim, N.WZ_KV_E4M3 if quantised else N.WZ_KV_BF16)
        self._desc = d
        self._ref = ctypes.byref(d)
        lib = N.lib()
        self._entry = {n: getattr(lib, n) for n in ("wz_paged_kv_write", "wz_paged_attn", "wz_paged_evict")}
        self._sizes = {}

    @classmethod
    def empty(cls, pages, page_size, kv_heads, head_dim, *, dtype=torch.bfloat16, shared=False, track=False,
              device="cuda"):
        """A cache over new pools; ``shared``: one row is K and V, ``track``: with weights and positions."""
        shape = (pages, kv_heads, page_size, head_dim)

        def pool():
            return torch.zeros(shape, dtype=torch.uint8, device=device).view(_E4M3) if dtype == _E4M3 else \
                torch.zeros(shape, dtype=dtype, device=device)

        def slots(dt=torch.float32):
            return torch.zeros(shape[:3], dtype=dt, device=device)

        q = dtype == _E4M3
        return cls(pool(), None if shared else pool(), k_scale=slots() if q else None,
                   v_scale=slots() if q and not shared else None, weights=slots() if track else None,
                   positions=slots(torch.int32) if track else None)

    # ---- checks (a decode step makes three calls for each layer: one pass over what can be wrong) ----

    def _ints(self, what, name, t, b):
        if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != b:
            raise ValueError(f"{what}: {name} must be int32 {[b]}, got {t.dtype} {list(t.shape)}")
        if t.device != self.device:
            raise ValueError(f"{what}: {name} is on {t.device}, the cache on {self.device}")
        return t if t.is_contiguous() else t.contiguous()

    def _table(self, what, t, b):
        if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != b:
            raise ValueError(f"{what}: table must be int32 [{b}, pages], got {t.dtype} {list(t.shape)}")
        if t.device != self.device:
            raise ValueError(f"{what}: table is on {t.device}, the cache on {self.device}")
        return t if t.is_contiguous() else t.contiguous()

    def _rows(self, what, name, t):
        """t as bf16 rows [.., .., .., D] that the kernels read in place: dense in their last dimension
        and 16-byte aligned (a view of a fused projection's output), else a copy."""
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{what}: bf16 {name} expected (got {t.dtype})")
        if t.device != self.device:
            raise ValueError(f"{what}: {name} is on {t.device}, the cache on {self.device}")
        sb, ss, sh, sd = t.stride()
        if sd != 1 or (sb | ss | sh | t.data_ptr() >> 1) & 7:
            t = t.clone(memory_format=torch.contiguous_format)
            sb, ss, sh, _ = t.stride()
        return t, _I64x3(sb, ss, sh)

    def _call(self, name, *args):
        index = self.device.index
        if _current_device() == index:
            rc = self._entry[name](self._ref, *args, _raw_stream(index))
        else:
            with torch.cuda.device(index):
                rc = self._entry[name](self._ref, *args, _raw_stream(index))
        if rc:
            N.check(rc, name)

    def _space(self, what, workspace, size, *shape):
        """The caller's workspace, or a new one of size(*shape) bytes."""
        if workspace is None:
            need = self._sizes.get(shape)
            if need is None:
                need = self._sizes[shape] = size(*shape)
            return torch.empty(need, dtype=torch.uint8, device=self.device)
        if workspace.dtype != torch.uint8 or workspace.device != self.device or not workspace.is_contiguous():
            raise ValueError(f"{what}: workspace must be a contiguous uint8 tensor on {self.device}")
        return workspace

    # ---- operators ----

    def write(self, k, v, table, start, count=None, position=None):
        """Puts new tokens into their pages: row i of k and v [b, s, kv_heads, head_dim] bf16 (v None where one
        row is both) goes to slot ``start[b] + i``, for i < ``count[b]`` (all s without it: a padded batch gives
        each sequence's own number).  An e4m3 cache quantises each row.  In a tracked cache a new slot has
        weight 0 and the position ``position[b] + i`` (its slot number without ``position``: give it once a
        cache has been cut).  Slots that the table has no page for are dropped.  A slot must be written once
        in a call."""
        shape = k.shape
        if len(shape) != 4 or shape[2] != self.kv_heads or shape[3] != self.head_dim:
            raise ValueError(f"PagedKV.write: k must be [b, s, {self.kv_heads}, {self.head_dim}], got {list(k.shape)}")
        if (v is None) != (self.v is None):
            raise ValueError("PagedKV.write: v is given where the cache has a v")
        if v is not None and v.shape != shape:
            raise ValueError(f"PagedKV.write: v {list(v.shape)} does not match k {list(k.shape)}")
        b, s = shape[0], shape[1]
        table = self._table("PagedKV.write", table, b)
        start = self._ints("PagedKV.write", "start", start, b)
        if count is not None:
            count = self._ints("PagedKV.write", "count", count, b)
        if position is not None:
            position = self._ints("PagedKV.write", "position", position, b)
        k, ks = self._rows("PagedKV.write", "k", k)
        v, vs = (None, None) if v is None else self._rows("PagedKV.write", "v", v)
        self._call("wz_paged_kv_write", k.data_ptr(), ks, N.ptr(v), vs, table.data_ptr(), table.shape[1],
                   start.data_ptr(), N.ptr(count), N.ptr(position), b, s)

    def attend(self, q, table, lens, softmax_scale, attn_sink=None, accumulate=False, out=None, workspace=None):
        """Attention of the s newest tokens of every sequence (1 to 16, already written) over its cached tokens:
        q [b, s, h, head_dim] bf16, ``lens`` [b] the tokens cached, the s new ones among them.  Query i of a
        sequence sees the slots below ``lens[b] - (s - 1 - i)``; query head j reads KV head j // (h / kv_heads).
        ``attn_sink`` [h] float32 adds a logit without a value to every row's sum, as in sparse_attn.  A row that
        sees nothing (a padded sequence of length 0) gives zeros.  -> [b, s, h, head_dim] bf16 (``out`` if given).

        ``accumulate`` adds to each slot's weight (a tracked cache) what the rows of its KV head gave it, in a
        fixed order.  ``out`` may not overlap q.  ``workspace``: a uint8 tensor of ``attend_workspace_bytes``, for
        calls that must not allocate; calls that overlap in time need one each."""
        if q.dim() != 4 or q.shape[3] != self.head_dim:
            raise ValueError(f"PagedKV.attend: q must be [b, s, h, {self.head_dim}], got {list(q.shape)}")
        b, s, h, d = q.shape
        table = self._table("PagedKV.attend", table, b)
        lens = self._ints("PagedKV.attend", "lens", lens, b)
        sink = None
        if attn_sink is not None:
            if attn_sink.shape != (h,) or attn_sink.dtype != torch.float32 or attn_sink.device != self.device:
                raise ValueError(f"PagedKV.attend: attn_sink must be float32 [{h}] on {self.device}")
            sink = attn_sink.contiguous()
        q, qs = self._rows("PagedKV.attend", "q", q)
        if out is None:
            out = torch.empty(b, s, h, d, dtype=torch.bfloat16, device=self.device)
        elif (out.shape != (b, s, h, d) or out.dtype != torch.bfloat16 or out.device != self.device
              or not out.is_contiguous()):
            raise ValueError(f"PagedKV.attend: out must be contiguous bf16 {[b, s, h, d]} on {self.device}")
        width = table.shape[1]
        workspace = self._space("PagedKV.attend", workspace, self.attend_workspace_bytes, b, s, h, width,
                                bool(accumulate))
        self._call("wz_paged_attn", q.data_ptr(), qs, N.ptr(sink), table.data_ptr(), width, lens.data_ptr(),
                   out.data_ptr(), b, s, h, float(softmax_scale), int(accumulate), workspace.data_ptr(),
                   workspace.numel())
        return out

    def attend_workspace_bytes(self, b, s, h, table_width, accumulate=False) -> int:
        """Device bytes of an ``attend`` call's partial results (and, accumulating, of its scores:
        4 b s h table_width page_size bytes)."""
        with torch.cuda.device(self.device):  # partials are counted by the compute units of the cache's device
            return int(N.lib().wz_paged_attn_workspace_bytes(self._ref, b, s, h, table_width, int(accumulate)))

    def evict(self, table, lens, keep, first=0, recent=0, out=None, workspace=None):
        """Cuts every sequence of a tracked cache to ``keep`` slots, in place and for each KV head by itself: the
        slots of positions below ``first``, the ``recent`` newest positions and then the slots of the highest
        weight stay (equal weights: the lower slot; NaN: the lowest).  The i-th dropped slot below ``keep`` takes
        over the i-th kept slot from ``keep`` on, with its rows, scales, weight and position, so nothing else
        moves and the pages past ``keep`` are free; slot order is no longer token order.  Slots that the table has
        no page for are neither kept nor filled: as many stay as have a page below ``keep``.  Sequences within the
        budget are left as they are.  -> min(lens, keep) int32 [b], in ``out`` if given (``lens`` itself may be, another view that
        overlaps it may not)."""
        keep, first, recent = int(keep), int(first), int(recent)
        if self.weights is None:
            raise ValueError("PagedKV.evict: the cache is not tracked (weights and positions)")
        b = lens.shape[0] if lens.dim() == 1 else -1
        table = self._table("PagedKV.evict", table, b)
        lens = self._ints("PagedKV.evict", "lens", lens, b)
        if out is None:
            out = torch.empty(b, dtype=torch.int32, device=self.device)
        elif self._ints("PagedKV.evict", "out", out, b) is not out:
            raise ValueError("PagedKV.evict: out must be contiguous")
        width = table.shape[1]
        workspace = self._space("PagedKV.evict", workspace, self.evict_workspace_bytes, b, width, keep)
        self._call("wz_paged_evict", table.data_ptr(), width, lens.data_ptr(), out.data_ptr(), b, keep, first, recent,
                   workspace.data_ptr(), workspace.numel())
        return out

    def evict_workspace_bytes(self, b, table_width, keep) -> int:
        """Device bytes of an ``evict`` call's lists of moves."""
        return int(N.lib().wz_paged_evict_workspace_bytes(self._ref, b, table_width, keep))
