"""Key / value cache of an attention layer in 8 bits, and the attention that reads it.

The reference keeps past keys and values in the model's type and concatenates (audiocraft/modules/transformer.py:266-298);
`LMModel` keeps them in one buffer of its `kv_dtype`.  This cache holds them in int8 with one scale for each block of 64 tokens
and head (include/acmi.h, acmi_kv8_cache): about half the bytes of a bf16 cache, which is what a decode step at a long context
reads.  `LMModel(kv_dtype=torch.int8)` runs its decode step on the same kernels.
"""
import typing as tp

import torch

from .. import _C

_DTYPES = (torch.float32, torch.bfloat16)


class KV8Cache:
    """`rows` streams of up to `capacity` tokens, `heads` key / value heads of `head_dim` features, of one layer.

    A row's newest block (64 tokens, partial or just completed) is held in `dtype` as stored; every block before it as int8 codes
    with a scale per block and head.  A block is quantised once, when its 64th token is stored.  A block that holds a NaN or an
    infinity reads back as NaN as a whole once it is quantised.

    How many tokens a row holds is the caller's: device int32 tensors `lens` / `start` [rows] are read by the kernels, so calls can
    be captured into a graph and replayed while the lengths advance on the device.  Lengths are not checked on the host: they are
    clamped to [0, capacity rounded up to whole blocks], and tokens past that are dropped.  Tokens of a row must be stored in
    order; rows that a call has no tokens for are left as they are.

    A call reads and writes the cache on the current stream, as any tensor operation does: calls on one cache from several
    streams need the caller's events between them; calls on different caches are independent (scratch belongs to a call).  Every call
    takes the process-wide `_C.device_lock`, like the models' device entries.
    """

    def __init__(self, rows: int, heads: int, head_dim: int, capacity: int, dtype: torch.dtype = torch.bfloat16,
                 device: tp.Union[str, torch.device] = 'cuda'):
        if dtype not in _DTYPES:
            raise ValueError(f"KV8Cache: dtype {dtype} (float32 or bfloat16)")
        if head_dim not in (16, 32, 64, 128):
            raise ValueError(f"KV8Cache: head_dim {head_dim} (16, 32, 64 or 128)")
        if not (0 < rows <= 65535 and 0 < heads <= 65535 and capacity > 0):
            raise ValueError(f"KV8Cache: rows {rows}, heads {heads}, capacity {capacity}")
        self.rows, self.heads, self.head_dim, self.dtype = rows, heads, head_dim, dtype
        self.blocks = -(-capacity // _C.KV8_BLOCK)
        if self.blocks >= 1 << 24:
            raise ValueError(f"KV8Cache: capacity {capacity} (at most {_C.KV8_BLOCK * ((1 << 24) - 1)})")
        self.capacity = self.blocks * _C.KV8_BLOCK
        if torch.device(device).type != 'cuda':
            raise ValueError(f"KV8Cache: device {device} (libacmi has no CPU fallback)")
        nb, blk = self.blocks, _C.KV8_BLOCK
        self.k_codes = torch.zeros(rows, heads, nb, blk, head_dim, device=device, dtype=torch.int8)
        self.v_codes = torch.zeros(rows, heads, nb, head_dim, blk, device=device, dtype=torch.int8)   # (tokens permuted: acmi.h)
        self.k_scale = torch.zeros(rows, heads, nb, device=device, dtype=torch.float32)
        self.v_scale = torch.zeros(rows, heads, nb, device=device, dtype=torch.float32)
        self.k_tail = torch.zeros(rows, heads, blk, head_dim, device=device, dtype=dtype)
        self.v_tail = torch.zeros(rows, heads, blk, head_dim, device=device, dtype=dtype)
        self.device = self.k_codes.device
        self._index, self._row_shape, self._work_floats = self.k_codes.get_device(), torch.Size((rows,)), {}
        self.desc = _C.KV8CacheDesc(self.k_codes.data_ptr(), self.v_codes.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(),
                                    self.k_tail.data_ptr(), self.v_tail.data_ptr(), _C.dtype_code(dtype), rows, heads, head_dim, nb)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.v_codes, self.k_scale, self.v_scale, self.k_tail, self.v_tail))

    def __reduce_ex__(self, protocol):   # (copy, deepcopy and pickle: `desc` would still name this cache's buffers)
        raise TypeError("KV8Cache: not copied as an object; store() what load() returned into a new one")

    # ------------------------------------------------------------------------------------- checks of arguments
    def _data(self, who: str, name: str, t: torch.Tensor, shape) -> torch.Tensor:
        if not isinstance(t, torch.Tensor) or t.shape != shape:
            raise ValueError(f"KV8Cache.{who}: {name} {tuple(getattr(t, 'shape', ()))}, expected {tuple(shape)}")
        return self._rows(who, name, t)

    def _rows(self, who: str, name: str, t: torch.Tensor) -> torch.Tensor:
        dt = t.dtype
        if (dt is not torch.float32 and dt is not torch.bfloat16) or t.get_device() != self._index:
            raise ValueError(f"KV8Cache.{who}: {name} is {dt} on {t.device}, expected float32 or bfloat16 on {self.device}")
        # the kernels read 16 bytes at a time: a view whose rows do not start on 16 bytes is copied
        st = t.stride()
        if st[-1] != 1 or (t.data_ptr() | (st[0] | st[1] | st[-2]) * (4 if dt is torch.float32 else 2)) & 15:
            t = t.clone(memory_format=torch.contiguous_format)
        return t

    def _words(self, who: str, name: str, t: tp.Optional[torch.Tensor], need: bool) -> tp.Optional[torch.Tensor]:
        if t is None and not need:
            return None
        if not isinstance(t, torch.Tensor) or t.shape != self._row_shape or t.dtype is not torch.int32 or t.get_device() != self._index:
            raise ValueError(f"KV8Cache.{who}: {name} must be int32 [{self.rows}] on {self.device}")
        return t if t.is_contiguous() else t.contiguous()

    def _work(self, S: int, Hq: int) -> int:
        n = self._work_floats.get((S, Hq))
        if n is None:
            cols = S * (Hq // self.heads)                   # query columns of a cache head, 64 to a workgroup
            if S > 1 << 20 or Hq > 65535 or cols > 1 << 21 or (-(-self.rows * self.heads // 8) * 8 * -(-cols // 64)) >= 1 << 24:
                raise ValueError(f"KV8Cache: {S} queries x {Hq} heads x {self.rows} rows in one call (2^20 queries, 65535 heads, 2^21 of both per "
                                 f"cache head, 2^24 groups of 64 in all)")
            n = self._work_floats[S, Hq] = _C.kv8_attn_work_floats(self.desc, S, Hq)
        return n

    # ------------------------------------------------------------------------------------- operators
    def store(self, k: torch.Tensor, v: torch.Tensor, start: tp.Optional[torch.Tensor] = None, n: tp.Optional[torch.Tensor] = None) -> None:
        """Keys and values [rows, L, heads, head_dim] of the tokens start[r] .. start[r] + n[r] - 1 of every row (n None: all L;
        start[r]: how many the row holds already, None: none).  Tokens past n[r] are padding and never read."""
        L = k.shape[1] if isinstance(k, torch.Tensor) and k.dim() == 4 else -1
        k = self._data('store', 'k', k, (self.rows, L, self.heads, self.head_dim))
        v = self._data('store', 'v', v, k.shape)
        if k.dtype != v.dtype:
            raise ValueError(f"KV8Cache.store: k is {k.dtype}, v is {v.dtype}")
        start, n = self._words('store', 'start', start, False), self._words('store', 'n', n, False)
        if L:
            with _C.device_lock:
                _C.kv8_store(self.desc, k, v, start, n)

    def load(self, lens: torch.Tensor, T: tp.Optional[int] = None, dtype: torch.dtype = torch.float32) -> tp.Tuple[torch.Tensor, torch.Tensor]:
        """The keys and values the cache holds, [rows, heads, T, head_dim] each (T None: the whole capacity), zeros past lens[r]."""
        lens = self._words('load', 'lens', lens, True)
        T = self.capacity if T is None else int(T)
        if not 0 <= T <= self.capacity or dtype not in _DTYPES:
            raise ValueError(f"KV8Cache.load: T {T} (0 .. {self.capacity}), dtype {dtype}")
        with _C.device_lock:
            k = torch.empty(self.rows, self.heads, T, self.head_dim, device=self.device, dtype=dtype)
            v = torch.empty_like(k)
            if T:
                _C.kv8_load(self.desc, lens, T, k, v)
        return k, v

    def decode(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor, past_context: int = 0,
               starts: tp.Optional[torch.Tensor] = None) -> torch.Tensor:
        """One new token per row: its key / value [rows, heads, head_dim] stored at position lens[r] and its queries
        [rows, G * heads, head_dim] attended over lens[r] + 1 tokens, in one launch (`lens` is not advanced).  past_context > 0:
        only the last past_context tokens before it are seen; starts [rows]: first token seen.  A row that is full (lens[r] at the
        capacity) drops the token and attends to what it holds.  -> like q, in q's dtype."""
        q, Hq = self._queries('decode', q, 3)
        k = self._data('decode', 'k', k, (self.rows, self.heads, self.head_dim))
        v = self._data('decode', 'v', v, k.shape)
        if k.dtype != v.dtype:
            raise ValueError(f"KV8Cache.decode: k is {k.dtype}, v is {v.dtype}")
        lens, starts = self._words('decode', 'lens', lens, True), self._words('decode', 'starts', starts, False)
        past, qs, work = self._past('decode', past_context), q.stride(), self._work(1, Hq)
        if (qs[0] | qs[1]) >> 31:                            # (few queries: strides in 32 bits)
            q = q.contiguous()
            qs = q.stride()
        with _C.device_lock:
            out = torch.empty(self.rows, Hq, self.head_dim, device=self.device, dtype=q.dtype)
            return _C.kv8_attn(self.desc, work, q, (qs[0], 0, qs[1]), 1, out, lens, 1, True, past, None, starts, k, v)

    def attend(self, q: torch.Tensor, lens: torch.Tensor, causal: bool = True, past_context: int = 0,
               q_lens: tp.Optional[torch.Tensor] = None, starts: tp.Optional[torch.Tensor] = None) -> torch.Tensor:
        """Queries [rows, S, G * heads, head_dim] over the lens[r] tokens a row holds (query head h reads head h // G).
        causal: a row's q_lens[r] (None: S) queries are its newest tokens, query i at position lens[r] - q_lens[r] + i; with
        past_context > 0 each sees only that many tokens before itself.  Not causal: every query sees the whole row (the states of
        an encoder).  starts [rows]: first token seen.  A query that sees nothing, and queries past q_lens[r], give zeros.
        -> like q, in q's dtype."""
        q, Hq = self._queries('attend', q, 4)
        S = q.shape[1]
        past = self._past('attend', past_context)
        if past and not causal:
            raise ValueError("KV8Cache.attend: past_context needs causal=True")
        lens, starts = self._words('attend', 'lens', lens, True), self._words('attend', 'starts', starts, False)
        q_lens = self._words('attend', 'q_lens', q_lens, False)
        work = self._work(S, Hq) if S else 0
        qs = q.stride()
        if (qs[0] | qs[1] | qs[2]) >> 31:                    # (few queries: strides in 32 bits)
            q = q.contiguous()
            qs = q.stride()
        with _C.device_lock:
            out = torch.empty(self.rows, S, Hq, self.head_dim, device=self.device, dtype=q.dtype)
            if S:
                _C.kv8_attn(self.desc, work, q, qs[:3], S, out, lens, 0, bool(causal), past, q_lens, starts)
        return out

    def _queries(self, who: str, q: torch.Tensor, dims: int) -> tp.Tuple[torch.Tensor, int]:
        sh = q.shape if isinstance(q, torch.Tensor) else ()
        if len(sh) != dims or sh[0] != self.rows or sh[-1] != self.head_dim or sh[-2] == 0 or sh[-2] % self.heads:
            raise ValueError(f"KV8Cache.{who}: q {tuple(sh)}: {dims} dimensions, {self.rows} rows, heads a multiple of {self.heads}, head_dim {self.head_dim}")
        return self._rows(who, 'q', q), sh[-2]

    def _past(self, who: str, past_context: tp.Optional[int]) -> int:
        past = int(past_context or 0)
        if past < 0:
            raise ValueError(f"KV8Cache.{who}: past_context {past}")
        return min(past, self.capacity)
