"""Python view of the paged Q4_0 cache (ctypes over include/bmo_attn.h): a pool
of pages, the plan that gives them to requests, appends, and the attention of
single tokens (``decode``) and ragged rows (``attend``) over them."""
from __future__ import annotations

from ._lib import lib
from .ring import RingError, _stream

_TYPES = {"float32": 0, "float16": 1, "bfloat16": 2, "uint8": 3, "int32": 4}  # (int32: lengths, tables, slots)
_CODES: dict = {}  # by dtype object (formatting one's name costs as much as a call)


def _code(x) -> int:
    code = _CODES.get(x.dtype)
    if code is None:
        code = _CODES[x.dtype] = _TYPES.get(str(x.dtype).rsplit(".", 1)[-1], 5)
    return code


def _type(x) -> int:
    """The element type (BMO_ATTN_F32 ..) of a tensor of rows or blocks."""
    code = _code(x)
    if code > 3:
        raise TypeError(f"expected a float32, float16, bfloat16 or uint8 tensor, got {x.dtype}")
    return code


class KVPages:
    """A device-resident pool of n_pages pages of page_size slots, for n_layers
    layers of n_kv_heads heads.

    The arrays that a request's pages live in are the caller's tensors (int32,
    on the pool's device): ``free`` [n_pages + 2], which ``list_init`` fills,
    ``table`` [n_batch][max_pages] and ``lens`` [n_batch], which ``plan`` keeps.
    A server's step plans the new tokens' slots once and then runs, per layer,
    ``append`` and ``attend`` for prompts or ``append_decode`` for single tokens
    (with the plan's ``status``, and ``n_new``, so that entries that it refused
    keep what they have and get zeros); the calls run on ``stream`` and can be captured in a
    HIP graph.  For cross attention the encoder's K and V are appended once, and
    ``attend`` with ``causal=False`` (or ``decode``) reads them."""

    def __init__(self, n_layers: int, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int):
        L = lib()
        h = L.bmo_kv_pages_create(n_layers, n_pages, page_size, n_kv_heads, head_dim)
        if not h:
            err = L.bmo_kv_pages_last_error(None)
            raise RuntimeError(f"bmo_kv_pages_create failed: {err.decode() if err else 'unknown'}")
        self._h = h
        self._free = L.bmo_kv_pages_free  # (__del__ needs no module globals)
        self._device = L.bmo_kv_pages_device(h)
        self.n_layers = n_layers
        self.n_pages = n_pages
        self.page_size = page_size
        self.n_kv_heads = n_kv_heads
        self.head_dim = head_dim

    # -- lifetime ---------------------------------------------------------------
    def close(self) -> None:
        h = getattr(self, "_h", None)
        if h:
            self._h = None
            self._free(h)

    def __del__(self):
        try:
            self.close()
        except Exception:  # interpreter teardown: nothing left to report to
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def handle(self) -> int:
        return self._h

    @property
    def nbytes(self) -> int:
        return int(lib().bmo_kv_pages_bytes(self._h))

    def last_error(self) -> str | None:
        e = lib().bmo_kv_pages_last_error(self._h)
        return e.decode() if e else None

    def _check(self, fn: str, rc: int) -> None:
        if rc != 0:
            raise RingError(fn, rc, self.last_error())

    # -- arguments --------------------------------------------------------------
    def _at(self, x, what: str) -> int:
        """Address of a tensor of the pool's device."""
        if x.get_device() != self._device:
            raise ValueError(f"{what} must be on the pool's device ({self._device}), not on {x.device}")
        return x.data_ptr()

    def _ints(self, x, what: str, n: int | None = None) -> int | None:
        """Address of a dense int32 tensor (of n elements), or None."""
        if x is None:
            return None
        if _code(x) != 4 or not x.is_contiguous() or (n is not None and x.numel() != n):
            size = "" if n is None else f" of {n} elements"
            raise ValueError(f"{what} must be a contiguous int32 tensor{size}")
        return x.data_ptr() if x.get_device() == self._device else self._at(x, what)

    def _rows(self, x, heads: int | None, what: str):
        """(address, stride, type, heads, tokens) of rows [tokens][heads][head_dim]."""
        shape = x.shape
        if len(shape) != 3 or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise ValueError(f"{what} must be [tokens][{heads or 'heads'}][{self.head_dim}], got {tuple(shape)}")
        n, h, d = shape
        stride = x.stride()
        if n and (stride[2] != 1 or (h > 1 and stride[1] != d)):
            raise ValueError(f"{what}: a token's heads must be contiguous")
        if n > 1 and stride[0] < h * d:
            raise ValueError(f"{what}: rows must not overlap (an expanded tensor)")
        at = x.data_ptr() if x.get_device() == self._device else self._at(x, what)
        return at, stride[0] if n > 1 else 0, _type(x), h, n

    def _out(self, x, n: int, heads: int, type_: int):
        if x.shape != (n, heads, self.head_dim) or not x.is_contiguous() or _type(x) != type_:
            raise ValueError(f"out must be a contiguous [{n}][{heads}][{self.head_dim}] tensor of q's type")
        return self._at(x, "out")

    def _table(self, lens, table):
        n, shape = lens.numel(), table.shape
        if len(shape) != 2 or shape[0] != n:
            raise ValueError("table must be [n_batch][max_pages]")
        return n, self._ints(lens, "lens"), self._ints(table, "table"), shape[1]

    def _work(self, workspace):
        if workspace is None:
            return None, 0
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        return self._at(workspace, "workspace"), workspace.numel() * workspace.element_size()

    # -- plan -------------------------------------------------------------------
    def list_init(self, free, stream=None) -> None:
        """Makes free (int32 [n_pages + 2]) hold every page."""
        self._check("bmo_kv_pages_list_init", lib().bmo_kv_pages_list_init(
            self._h, self._ints(free, "free", self.n_pages + 2), _stream(stream)))

    def plan(self, free, n_new, lens, table, tok_start=None, slots=None, positions=None, entries=None, status=None,
             stream=None) -> None:
        """n_new[b] more (or, negative, fewer) positions for every entry: lens,
        table and free become the new state; slots, positions and entries
        [max_tok] tell the new tokens' places (append_decode needs none of them),
        tok_start [n_batch + 1] where an entry's tokens begin, status [n_batch] 0
        where it was done, 1 without pages, 2 out of range (or past max_tok)."""
        n, lens_p, table_p, width = self._table(lens, table)
        sizes = {x.numel() for x in (slots, positions, entries) if x is not None} or {2**31 - 1}
        if len(sizes) > 1:
            raise ValueError("slots, positions and entries must have the same size")
        self._check("bmo_kv_pages_plan", lib().bmo_kv_pages_plan(
            self._h, self._ints(free, "free", self.n_pages + 2), n, self._ints(n_new, "n_new", n), lens_p, table_p, width,
            self._ints(tok_start, "tok_start", n + 1), sizes.pop(), self._ints(slots, "slots"),
            self._ints(positions, "positions"), self._ints(entries, "entries"), self._ints(status, "status", n),
            _stream(stream)))

    # -- rows in and out ----------------------------------------------------------
    def _slots(self, fn: str, call, layer: int, slots, k, v, stream) -> None:
        n = slots.numel()
        if _type(k) == 3:  # ggml blocks
            shape = (n, self.n_kv_heads, self.head_dim // 32, 18)
            if tuple(k.shape) != shape or tuple(v.shape) != shape or not (k.is_contiguous() and v.is_contiguous()):
                raise ValueError(f"blocks must be contiguous uint8 {shape}")
            kp, vp, stride, type_, vtype = self._at(k, "k"), self._at(v, "v"), 0, 3, _type(v)
        else:
            kp, stride, type_, _, nk = self._rows(k, self.n_kv_heads, "k")
            vp, vstride, vtype, _, nv = self._rows(v, self.n_kv_heads, "v")
            if nk != n or nv != n or vstride != stride:
                raise ValueError("k and v must have one row a slot and the same stride")
        if vtype != type_:
            raise ValueError("k and v must have the same type")
        self._check(fn, call(self._h, int(layer), n, self._ints(slots, "slots"), type_, kp, vp, stride, _stream(stream)))

    def append(self, layer: int, slots, k, v, stream=None) -> None:
        """Quantizes rows k, v [n_tok][n_kv_heads][head_dim] (or copies uint8
        ggml blocks [n_tok][n_kv_heads][head_dim / 32][18]) into slots [n_tok]."""
        self._slots("bmo_kv_pages_append", lib().bmo_kv_pages_append, layer, slots, k, v, stream)

    def gather(self, layer: int, slots, k, v, stream=None) -> None:
        """What slots [n_tok] hold, into k and v (values, or uint8 blocks)."""
        self._slots("bmo_kv_pages_gather", lib().bmo_kv_pages_gather, layer, slots, k, v, stream)

    # -- attention ----------------------------------------------------------------
    def workspace_bytes(self, n_heads: int) -> int:
        """Bytes of a workspace for decode and attend with n_heads query heads;
        calls that may overlap need one each."""
        return int(lib().bmo_kv_pages_workspace_bytes(self._h, int(n_heads)))

    def decode(self, layer: int, lens, table, q, out, scale: float = 0.0, window: int = 0, max_len: int = 0,
               workspace=None, stream=None) -> None:
        """One row per entry over its last min(len, window) positions (window 0:
        all): q and out [n_batch][n_heads][head_dim]."""
        n, lens_p, table_p, width = self._table(lens, table)
        qp, stride, type_, heads, nq = self._rows(q, None, "q")
        if nq != n:
            raise ValueError("q must have one row an entry")
        self._check("bmo_kv_pages_decode", lib().bmo_kv_pages_decode(
            self._h, int(layer), n, lens_p, table_p, width, heads, type_, qp, stride, self._out(out, n, heads, type_),
            float(scale), int(window), int(max_len), *self._work(workspace), _stream(stream)))

    def append_decode(self, layer: int, lens, table, q, k, v, out, scale: float = 0.0, window: int = 0,
                      max_len: int = 0, workspace=None, stream=None, n_new=None, status=None) -> None:
        """decode with k and v [n_batch][n_kv_heads][head_dim] appended at each
        entry's last position (lens counts it already).  With the n_new and
        status [n_batch] of the plan before, entries that it did not let grow are
        left as they are and get zeros; without them every entry with positions
        must have grown."""
        n, lens_p, table_p, width = self._table(lens, table)
        qp, stride, type_, heads, nq = self._rows(q, None, "q")
        kp, kstride, ktype, _, nk = self._rows(k, self.n_kv_heads, "k")
        vp, vstride, vtype, _, nv = self._rows(v, self.n_kv_heads, "v")
        if nq != n or nk != n or nv != n or kstride != vstride or ktype != type_ or vtype != type_:
            raise ValueError("q, k and v must have one row an entry and one type, k and v the same stride")
        fn, granted = "bmo_kv_pages_append_decode", ()
        if n_new is not None or status is not None:
            if n_new is None or status is None:
                raise ValueError("n_new and status come together")
            fn, granted = fn + "_granted", (self._ints(n_new, "n_new", n), self._ints(status, "status", n))
        self._check(fn, getattr(lib(), fn)(
            self._h, int(layer), n, *granted, lens_p, table_p, width, heads, type_, qp, stride, kp, vp, kstride,
            self._out(out, n, heads, type_), float(scale), int(window), int(max_len), *self._work(workspace),
            _stream(stream)))

    def attend(self, layer: int, q_start, lens, table, q, out, causal: bool = True, scale: float = 0.0,
               window: int = 0, max_rows: int = 0, max_len: int = 0, workspace=None, stream=None,
               status=None) -> None:
        """Ragged rows q and out [n_rows][n_heads][head_dim] (fp16 or bf16), entry
        b's from q_start[b] to q_start[b + 1]: its last positions (causal), or
        rows that see all of its positions (cross attention).  With the status
        [n_batch] of the plan before, rows of entries that it refused are zeros."""
        n, lens_p, table_p, width = self._table(lens, table)
        qp, stride, type_, heads, rows = self._rows(q, None, "q")
        fn, granted = "bmo_kv_pages_attend", ()
        if status is not None:
            fn, granted = fn + "_granted", (self._ints(status, "status", n),)
        self._check(fn, getattr(lib(), fn)(
            self._h, int(layer), n, *granted, self._ints(q_start, "q_start", n + 1), lens_p, table_p, width, rows, heads, type_, qp,
            stride, self._out(out, rows, heads, type_), float(scale), int(bool(causal)), int(window), int(max_rows),
            int(max_len), *self._work(workspace), _stream(stream)))
