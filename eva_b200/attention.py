"""Attention between the MoE layers: rotary positions, a paged 8-bit key/value cache, and causal attention over it.

* `Rotary` rotates part of each head by its token's position (interleaved or half layout, linear, NTK or YaRN scaling).
* `PagedKVCache` holds one layer's keys and values as e4m3 codes with a power-of-two scale for each 16 tokens and head;
  `append` rotates, quantises and writes new tokens, `attend` reads them.
* `PagedBatch` names the sequences of a step: which token rows, how long, and which pages.
* `PagedAttention` is the attention half of a layer (projections around the three), which `MoEStack` calls.

The reference's attention (runtime/ds41/model.py:566-937 `Attention`) reads a 4-bit compressed cache through an index;
this is plain causal attention, for layers of DeepSeek shape without that index. Everything runs on the caller's current
CUDA stream and never synchronises the host, so it can be captured in a CUDA graph and replayed; outputs and
workspaces come from torch's allocator for each call. No gradients are recorded (of the rotation, apply(inverse=True) is one):
tensors that require them are refused unless gradients are off, and so are dual tensors of forward-mode differentiation.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import torch
from torch.autograd import forward_ad as _forward

from . import _lib

_F16, _BF16, _F32, _I32, _I64 = torch.float16, torch.bfloat16, torch.float32, torch.int32, torch.int64
_E4M3, _E8M0, _U8 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.uint8
_DTYPE = {_F16: _lib.DTYPE_F16, _BF16: _lib.DTYPE_BF16, _F32: _lib.DTYPE_F32}
PAGE, BLOCK = _lib.KV_PAGE, _lib.KV_BLOCK
HEAD_DIMS = ((64, 64), (128, 128), (192, 128))
_INT32_MAX = 2**31 - 1
_DECODE_ROWS = 16   # of the library: rows that share a key and value, up to which the decode kernel takes a call


def _device(device) -> torch.device:
    device = torch.device(device)
    if device.type != "cuda" or not torch.cuda.is_available():
        raise RuntimeError("the attention operators require a CUDA device; there is no CPU fallback")
    return torch.device("cuda", torch.cuda.current_device()) if device.index is None else device


_HERE = contextlib.nullcontext()


def _on(device):
    """The library launches on the current device: make it the tensors'."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


if hasattr(torch._C, "_cuda_getCurrentRawStream"):   # the same handle without a Stream object (2 us less a call)
    def _stream(device):   # noqa: F811
        return torch._C._cuda_getCurrentRawStream(device.index)


def _rows(t, name, device, dtypes, heads=None, dim=None):
    if not isinstance(t, torch.Tensor) or t.device != device or t.ndim != 3 or t.dtype not in dtypes:
        raise ValueError(f"{name} must be [tokens, heads, dim] of {', '.join(map(str, dtypes))} on {device}")
    if (heads is not None and t.shape[1] != heads) or (dim is not None and t.shape[2] != dim):
        raise ValueError(f"{name} must be [tokens, {'heads' if heads is None else heads}, {dim}]")
    return t


class Rotary:
    """Rotation of `dim` dimensions of a head from `offset` on by position * frequency_i, i < dim / 2.

    layout: "half" pairs dimension i with i + dim / 2, "interleaved" 2i with 2i + 1. Frequencies are
    base^(-2i / dim), changed by `scaling`: "linear" divides positions by `factor`; "ntk" raises the base to
    base * factor^(dim / (dim - 2)); "yarn" divides the frequencies that turn less than beta_slow times in
    original_len positions by `factor`, keeps those above beta_fast, goes linearly between, and scales the result by
    0.1 ln(factor) + 1. mscale replaces that scale. Angles are exact modulo a turn at any position."""

    def __init__(self, dim, *, base=10000.0, layout="interleaved", offset=0, scaling="none", factor=1.0,
                 original_len=4096, beta_fast=32.0, beta_slow=1.0, mscale=None, device="cuda"):
        self.inv_freq, scale = rotary_frequencies(dim, base=base, scaling=scaling, factor=factor,
                                                  original_len=original_len, beta_fast=beta_fast, beta_slow=beta_slow)
        if layout not in ("half", "interleaved"):
            raise ValueError("layout must be 'half' or 'interleaved'")
        if type(offset) is not int or offset < 0 or offset % 2:
            raise ValueError("offset must be an even nonnegative int")
        mscale = scale if mscale is None else mscale
        if not isinstance(mscale, (int, float)) or not math.isfinite(mscale):
            raise ValueError("mscale must be a finite number")
        self.dim, self.offset, self.layout, self.mscale = dim, offset, layout, float(mscale)
        self.device = _device(device)
        self.lib = _lib.load()
        self.turns = torch.tensor(turns_of(self.inv_freq), dtype=_I64, device=self.device)
        args = (dim, offset, int(layout == "interleaved"))
        self._c = _lib.EvaRotary(*args, 0, self.mscale, 0, self.turns.data_ptr())
        self._c_inverse = _lib.EvaRotary(*args, 1, self.mscale, 0, self.turns.data_ptr())
        self._ref, self._ref_inverse = ctypes.byref(self._c), ctypes.byref(self._c_inverse)
        self._pairs, self._end = layout == "interleaved", offset + dim

    def apply(self, x, positions, *, inverse=False, out=None):
        """x [tokens, heads, head_dim] (BF16, Half or Float; last dimension contiguous) rotated by positions (int32 or
        int64 [tokens]); inverse rotates back by the same scale, as the gradient does. out: x itself, or a tensor that does not
        overlap it; default a new one."""
        device = self.device
        if not isinstance(x, torch.Tensor) or x.ndim != 3 or x.dtype not in _DTYPE or x.device != device:
            raise ValueError(f"x must be [tokens, heads, head_dim] of BF16, Half or Float on {device}")
        tokens, heads, head_dim = x.shape
        if self._end > head_dim:
            raise ValueError(f"x's heads have {head_dim} dimensions, the rotation ends at {self._end}")
        if heads < 1:
            raise ValueError("x has no heads")
        if (not isinstance(positions, torch.Tensor) or positions.ndim != 1 or positions.shape[0] != tokens
                or positions.dtype not in (_I64, _I32) or positions.device != device or not positions.is_contiguous()):
            raise ValueError(f"positions must be contiguous int32 or int64 [{tokens}] on {device}")
        if x.requires_grad or _forward._current_level >= 0:
            _no_grad(x)
        src = x if tokens == 0 else self._movable(x, out is x)
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
        elif out is not x:
            src = self._check_out(x, src, out)
        elif _folded(x):
            raise ValueError("in place, x must not overlap itself")
        if tokens == 0:
            return out
        if src is None:
            raise ValueError("the kernel cannot move this x or out: it needs whole interleaved pairs and, of what it writes to, "
                             "a contiguous last dimension")
        xt, xh, _ = src.stride()
        ot, oh, _ = out.stride()
        if tokens == 1:
            xt = ot = 0
        if heads == 1:
            xh = oh = 0
        with _on(device):
            rc = self.lib.eva_rotary(self._ref_inverse if inverse else self._ref, src.data_ptr(), _DTYPE[x.dtype], tokens, heads,
                                     head_dim, xt, xh, positions.data_ptr(), positions.dtype == _I64, out.data_ptr(), ot, oh,
                                     _stream(device))
        if rc:
            _lib.check(rc, "eva_rotary")
        return out

    def _check_out(self, x, src, out):
        """What to rotate from (x, or a copy of it) into a given out that is not x; None where the kernel cannot write to out."""
        _rows(out, "out", self.device, (x.dtype,), x.shape[1], x.shape[2])
        if out.shape[0] != x.shape[0]:
            raise ValueError("out must have x's shape")
        if out.requires_grad or _forward._current_level >= 0:
            _no_grad(out)
        if _folded(out):
            raise ValueError("out must not overlap itself")
        same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride()   # the same memory: in place
        if not same and _overlap(x, out):
            raise ValueError("out must be x itself or not overlap it")
        if x.shape[0] == 0:
            return x
        if self._movable(out, True) is None or (same and src is not x):
            return None
        return src

    def _movable(self, t, must):
        """t, or a contiguous copy of it (None where it must be t itself), as the kernel moves it: whole elements side by side,
        interleaved pairs at addresses that are multiples of a pair."""
        st, sh, sd = t.stride()
        n, h, d = t.shape
        if sd == 1 or d == 1:
            if not self._pairs:
                return t
            if (t.data_ptr() % (2 * t.element_size()) == 0 and d % 2 == 0 and (st % 2 == 0 or n == 1) and (sh % 2 == 0 or h == 1)):
                return t
        if must or (self._pairs and d % 2):
            return None
        return t.clone(memory_format=torch.contiguous_format)


def _span(t):
    n = t.element_size()
    return t.data_ptr(), t.data_ptr() + n * (1 + sum((s - 1) * st for s, st in zip(t.shape, t.stride())))


def _no_grad(*tensors):
    """The operators record no gradients: a call that autograd would follow is refused, not answered without one. Tangents of
    forward mode are followed under no_grad too."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError("the attention operators record no gradients: call them under torch.no_grad()")
    if any(_dual(t) for t in tensors):
        raise ValueError("the attention operators have no forward-mode derivatives: unpack dual tensors first")


def _dual(t):
    return _forward._current_level >= 0 and _forward.unpack_dual(t).tangent is not None


def _folded(t):
    """Whether two elements of t may share memory."""
    end = 0
    for st, n in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1):
        if st <= end:
            return True
        end += (n - 1) * st
    return False


def _overlap(a, b):
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a0 < b1 and b0 < a1


def rotary_frequencies(dim, *, base=10000.0, scaling="none", factor=1.0, original_len=4096, beta_fast=32.0, beta_slow=1.0):
    """(angle per position of each pair, scale of the rotated part), as Python floats."""
    if type(dim) is not int or dim < 2 or dim % 2:
        raise ValueError("dim must be an even positive int")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise ValueError("scaling must be 'none', 'linear', 'ntk' or 'yarn'")
    if not (math.isfinite(base) and base > 1.0 and math.isfinite(factor) and factor >= 1.0):
        raise ValueError("base must be above 1 and factor at least 1")
    if scaling == "ntk":
        if dim < 4:
            raise ValueError("ntk scaling needs dim >= 4")
        base = base * factor ** (dim / (dim - 2))
    freq = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        return [f / factor for f in freq], 1.0
    if scaling != "yarn":
        return freq, 1.0
    if not (original_len >= 1 and beta_fast >= beta_slow > 0):
        raise ValueError("yarn needs original_len >= 1 and beta_fast >= beta_slow > 0")

    def pair_turning(times):   # the (fractional) pair that makes so many turns in original_len positions
        return dim * math.log(original_len / (times * 2 * math.pi)) / (2 * math.log(base))

    low = max(math.floor(pair_turning(beta_fast)), 0)
    high = min(math.ceil(pair_turning(beta_slow)), dim - 1)
    width = max(high - low, 0.001)
    out = []
    for i, f in enumerate(freq):
        slow = min(max((i - low) / width, 0.0), 1.0)
        out.append(f / factor * slow + f * (1.0 - slow))
    return out, 0.1 * math.log(factor) + 1.0


def turns_of(inv_freq):
    """Frequencies as fractions of a turn times 2^64, modulo 2^64, as int64 values (the same bits)."""
    out = []
    for f in inv_freq:
        t = f / (2 * math.pi)
        t = int((t - math.floor(t)) * 2.0**64) % 2**64
        out.append(t - 2**64 if t >= 2**63 else t)
    return out


class PagedBatch:
    """The sequences of one step. q_start: int32 [seqs + 1], sequence b has token rows q_start[b] .. q_start[b + 1] - 1 of the
    step's tensors; they are the last ones of its seq_lens[b] tokens (int32 [seqs], new ones included), and token t of it
    lies in page table[b, t // 64] (int32 [seqs, pages], contiguous rows). max_q: the most rows of a sequence.

    The tensors stay the caller's: a captured step is replayed with new contents in them (max_q and the table's width
    bound what they may hold). A padding sequence has length 0 (its rows come out zero, nothing is appended). What does
    not fit (page ids outside the cache, lengths beyond the table, rows out of order) sets STATUS_BAD_BATCH in the cache's
    status and is left out. To a sequence without rows an append does nothing: its pages may be another's. A page that stands twice among those that one call appends to (of two sequences, or of one) is the
    caller's error: its contents are then undefined."""

    def __init__(self, q_start, seq_lens, table, max_q):
        for name, t, nd in (("q_start", q_start, 1), ("seq_lens", seq_lens, 1), ("table", table, 2)):
            if not isinstance(t, torch.Tensor) or t.dtype != _I32 or t.ndim != nd or t.device.type != "cuda":
                raise ValueError(f"{name} must be an int32 CUDA tensor of {nd} dimension(s)")
            if t.device != q_start.device:
                raise ValueError("q_start, seq_lens and table must be on one device")
            if t.numel() > 1 and t.stride(-1) != 1 and t.shape[-1] > 1:
                raise ValueError(f"{name} must be contiguous in its last dimension")
        self.seqs = seq_lens.shape[0]
        if q_start.shape[0] != self.seqs + 1 or table.shape[0] != self.seqs:
            raise ValueError("q_start must be [seqs + 1] and table [seqs, pages]")
        if type(max_q) is not int or not 0 <= max_q <= 1 << 28:
            raise ValueError("max_q must be a nonnegative int")
        if self.seqs > 1 << 24 or table.shape[1] > 1 << 24 or (self.seqs and table.shape[1] < 1):
            raise ValueError("at most 2^24 sequences, and 1 to 2^24 pages of one")
        self.q_start, self.seq_lens, self.table, self.max_q = q_start, seq_lens, table, max_q
        self.device = q_start.device
        stride = table.stride(0) if self.seqs > 1 else table.shape[1]
        if stride < 0 or (self.seqs > 1 and stride < table.shape[1]):
            raise ValueError("table rows must not overlap")
        self._c = _lib.EvaKvBatch(self.seqs, 0, max_q, table.shape[1], stride, q_start.data_ptr(), seq_lens.data_ptr(),
                                  table.data_ptr())
        self._refs = {}

    def _for(self, tokens):
        """The C struct of a step of so many token rows."""
        ref = self._refs.get(tokens)
        if ref is None:
            if tokens > _INT32_MAX:
                raise ValueError("too many token rows")
            if tokens and self.seqs and not self.max_q:
                raise ValueError("a batch with max_q 0 has no token rows")
            if len(self._refs) > 64:
                self._refs.clear()
            c = self._c
            ref = ctypes.byref(_lib.EvaKvBatch(c.seqs, tokens, c.max_q, c.max_pages, c.table_stride, c.q_start, c.seq_lens, c.table))
            self._refs[tokens] = ref
        return ref


class PagedKVCache:
    """One layer's keys and values in pages of 64 tokens, 8 bits each: codes e4m3, one scale 2^e (E8M0) for each 16 tokens
    and head. (key_dim, value_dim) is (64, 64), (128, 128) or (192, 128).

    k [pages, kv_heads, 64, key_dim], v [pages, kv_heads, value_dim, 64] (a dimension's tokens side by side), k_scale and
    v_scale [pages, kv_heads, 4]; existing contiguous tensors may be given (float8 or uint8; scale bytes 1 .. 253, and no NaN among the
    value codes of a sequence's tokens: it would reach rows that do not see its token; an append writes none)."""

    def __init__(self, pages, kv_heads, key_dim, value_dim=None, *, device="cuda", k=None, v=None, k_scale=None, v_scale=None):
        value_dim = key_dim if value_dim is None else value_dim
        if (key_dim, value_dim) not in HEAD_DIMS:
            raise ValueError(f"(key_dim, value_dim) must be one of {HEAD_DIMS}")
        if type(pages) is not int or type(kv_heads) is not int or not 1 <= pages <= _INT32_MAX or not 1 <= kv_heads <= 65535:
            raise ValueError("pages must be a positive int and kv_heads one in 1..65535")
        self.device = _device(device)
        self.lib = _lib.load()
        self.pages, self.kv_heads, self.key_dim, self.value_dim = pages, kv_heads, key_dim, value_dim
        self.k = self._buffer(k, (pages, kv_heads, PAGE, key_dim), _E4M3, "k")
        self.v = self._buffer(v, (pages, kv_heads, value_dim, PAGE), _E4M3, "v")
        self.k_scale = self._buffer(k_scale, (pages, kv_heads, PAGE // BLOCK), _E8M0, "k_scale")
        self.v_scale = self._buffer(v_scale, (pages, kv_heads, PAGE // BLOCK), _E8M0, "v_scale")
        self._status = torch.zeros(1, dtype=_I32, device=self.device)
        self._c = _lib.EvaKvCache(pages, kv_heads, key_dim, value_dim, self.k.data_ptr(), self.v.data_ptr(),
                                  self.k_scale.data_ptr(), self.v_scale.data_ptr(), self._status.data_ptr())
        self._ref = ctypes.byref(self._c)
        self._scale, self._sizes = key_dim ** -0.5, {}   # default scale; workspace bytes by rows that share a key

    def _buffer(self, t, shape, dtype, name):
        if t is None:
            return torch.zeros(shape, dtype=_U8, device=self.device).view(dtype)
        if (not isinstance(t, torch.Tensor) or t.device != self.device or tuple(t.shape) != shape or t.dtype not in (dtype, _U8)
                or not t.is_contiguous() or t.data_ptr() % 16):
            raise ValueError(f"{name} must be a contiguous {dtype} or uint8 {list(shape)} on {self.device}, 16-byte aligned")
        return t.view(dtype)

    def _batch(self, batch, tokens):
        if not isinstance(batch, PagedBatch) or batch.device != self.device:
            raise ValueError(f"batch must be a PagedBatch on {self.device}")
        return batch._for(tokens)

    def append(self, k, v, batch, *, rotary=None):
        """Write the batch's new tokens: k [tokens, kv_heads, key_dim] rotated by each token's position in its sequence, and
        v [tokens, kv_heads, value_dim] (BF16 or Half, any token and head strides), quantised. A block's scale is the smallest
        power of two that fits its tokens; one that a later token raises has its older codes rescaled. A token with a
        non-finite element (of the rotated key too) gets a NaN key: the rows that see it become NaN, and no others."""
        device = self.device
        if (not isinstance(k, torch.Tensor) or k.ndim != 3 or k.dtype not in (_BF16, _F16) or k.device != device
                or k.shape[1] != self.kv_heads or k.shape[2] != self.key_dim):
            raise ValueError(f"k must be BF16 or Half [tokens, {self.kv_heads}, {self.key_dim}] on {device}")
        tokens = k.shape[0]
        if (not isinstance(v, torch.Tensor) or v.ndim != 3 or v.dtype != k.dtype or v.device != device
                or v.shape != (tokens, self.kv_heads, self.value_dim)):
            raise ValueError(f"v must be {k.dtype} [{tokens}, {self.kv_heads}, {self.value_dim}] on {device}")
        if rotary is not None:
            if not isinstance(rotary, Rotary) or rotary.device != device:
                raise ValueError(f"rotary must be a Rotary on {device}")
            if rotary._end > self.key_dim:
                raise ValueError(f"the rotation ends at {rotary._end}, keys have {self.key_dim} dimensions")
        if k.requires_grad or v.requires_grad or _forward._current_level >= 0:
            _no_grad(k, v)
        b = self._batch(batch, tokens)
        if k.stride(2) != 1:
            k = k.contiguous()
        if v.stride(2) != 1:
            v = v.contiguous()
        (kt, kh, _), (vt, vh, _) = k.stride(), v.stride()
        with _on(device):
            rc = self.lib.eva_kv_append(self._ref, b, None if rotary is None else rotary._ref, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh,
                                        _DTYPE[k.dtype], _stream(device))
        if rc:
            _lib.check(rc, "eva_kv_append")

    def attend(self, q, batch, *, scale=None, window=0, out=None):
        """softmax(scale q k^T) v of q [tokens, heads, key_dim] (BF16 or Half, already rotated) over the batch's sequences,
        new tokens included: a row sees the tokens up to its own position, with window > 0 the last `window` of them.
        heads is a multiple of kv_heads. Returns [tokens, heads, value_dim] of q's type; rows that see nothing are zero, rows behind
        the last sequence, and of one that does not fit, are left as they were (in out; a new tensor has no values there).

        Values below 2^-39, and weights (times their block's value scale) below 2^-28 of a row's largest, may count as zero in the
        output (not in the softmax's sum); with values above 2^43 beside much smaller ones the sum may lose tokens. Scores count as 32-bit floats: one above
        their range makes its row NaN, one below has no weight."""
        device = self.device
        if (not isinstance(q, torch.Tensor) or q.ndim != 3 or q.dtype not in (_BF16, _F16) or q.device != device
                or q.shape[2] != self.key_dim):
            raise ValueError(f"q must be BF16 or Half [tokens, heads, {self.key_dim}] on {device}")
        tokens, heads, _ = q.shape
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"heads must be a multiple of {self.kv_heads}")
        if type(window) is not int or not 0 <= window <= _INT32_MAX:
            raise ValueError("window must be a nonnegative int")
        if scale is None:
            scale = self._scale
        elif not isinstance(scale, (int, float)) or not 0 <= scale <= 2e38:
            raise ValueError("scale must be a finite nonnegative number")
        if q.requires_grad or _forward._current_level >= 0:
            _no_grad(q)
        b = self._batch(batch, tokens)
        st, sh, sd = q.stride()
        if tokens == 1:
            st = 0
        if heads == 1:
            sh = 0
        if sd != 1 or st % 8 or sh % 8 or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
            st, sh, _ = q.stride()
        if out is None:
            out = q.new_empty((tokens, heads, self.value_dim))
        elif (not isinstance(out, torch.Tensor) or out.device != device or out.dtype != q.dtype or not out.is_contiguous()
              or out.shape != (tokens, heads, self.value_dim) or out.data_ptr() % 16):
            raise ValueError(f"out must be a contiguous {q.dtype} [{tokens}, {heads}, {self.value_dim}] on {device}, 16-byte aligned")
        else:
            if _overlap(q, out):
                raise ValueError("out must not overlap q")
            if out.requires_grad or _forward._current_level >= 0:
                _no_grad(out)
        rows = min(batch.max_q * (heads // self.kv_heads), _DECODE_ROWS + 1)   # above them the size is the same
        n = self._sizes.get(rows)
        with _on(device):
            if n is None:
                n = self.lib.eva_kv_attend_workspace(self._ref, b, heads)
                if n == 0:
                    raise ValueError("unsupported batch")
                self._sizes[rows] = n
            ws = q.new_empty((n,), dtype=_U8)
            rc = self.lib.eva_kv_attend(self._ref, b, q.data_ptr(), _DTYPE[q.dtype], heads, st, sh, scale, window, ws.data_ptr(), n,
                                        out.data_ptr(), _stream(device))
        if rc:
            _lib.check(rc, "eva_kv_attend")
        return out

    def values(self, pages):
        """The keys [n, kv_heads, 64, key_dim] and values [n, kv_heads, 64, value_dim] that the pages (int64 [n]) hold, as floats."""
        k = self.k[pages].to(_F32) * self.k_scale[pages].to(_F32).repeat_interleave(BLOCK, -1)[..., None]
        v = self.v[pages].to(_F32) * self.v_scale[pages].to(_F32).repeat_interleave(BLOCK, -1)[..., None, :]
        return k, v.transpose(2, 3)

    def status(self) -> int:
        """The device status bits (reads them back: synchronises the host). They stay until clear_status(), whatever later calls do."""
        return int(self._status.item())

    def clear_status(self) -> None:
        self._status.zero_()


class PagedAttention:
    """The attention half of a layer: query, key and value projections, rotation, append, attention, output projection.

    wqkv: BF16 [heads * key_dim + kv_heads * (key_dim + value_dim), hidden] (queries, keys, values, one below the other),
    wo: BF16 [hidden, heads * value_dim]; the cache and the rotation are the layer's own (or shared, for the rotation). The
    projections are plain matrix products; keys and values go to the cache as they lie in the projection's rows."""

    def __init__(self, cache, wqkv, wo, heads, rotary=None, *, scale=None, window=0):
        if not isinstance(cache, PagedKVCache):
            raise ValueError("cache must be a PagedKVCache")
        if type(heads) is not int or heads < 1 or heads % cache.kv_heads:
            raise ValueError(f"heads must be a multiple of {cache.kv_heads}")
        rows = heads * cache.key_dim + cache.kv_heads * (cache.key_dim + cache.value_dim)
        for name, w, shape in (("wqkv", wqkv, (rows, None)), ("wo", wo, (None, heads * cache.value_dim))):
            if (not isinstance(w, torch.Tensor) or w.dtype != _BF16 or w.ndim != 2 or w.device != cache.device
                    or any(n is not None and n != m for n, m in zip(shape, w.shape))):
                raise ValueError(f"{name} must be BF16 {['hidden' if n is None else n for n in shape]} on {cache.device}")
        if wqkv.shape[1] != wo.shape[0]:
            raise ValueError("wqkv and wo must have the same hidden size")
        if rotary is not None and not isinstance(rotary, Rotary):
            raise ValueError("rotary must be a Rotary")
        self.cache, self.wqkv, self.wo, self.heads, self.rotary = cache, wqkv, wo, heads, rotary
        self.scale, self.window, self.hidden = scale, window, wqkv.shape[1]

    def forward(self, h, batch, positions, *, out_f32=None):
        """h: BF16 [tokens, hidden], the batch's new tokens; positions: int32 or int64 [tokens], each token's place in its
        sequence. Returns BF16 [tokens, hidden], or FP32 in out_f32 where that is given, not rounded to BF16 in between. Rows of no sequence (behind the last one,
        or of one that does not fit the batch) are zero."""
        c = self.cache
        if h.ndim != 2 or h.shape[1] != self.hidden or h.dtype != _BF16 or h.device != c.device:
            raise ValueError(f"h must be BF16 [tokens, {self.hidden}] on {c.device}")
        if out_f32 is not None and (out_f32.shape != h.shape or out_f32.dtype != _F32 or out_f32.device != c.device):
            raise ValueError(f"out_f32 must be FP32 {list(h.shape)} on {c.device}")
        rows = h @ self.wqkv.T
        nq, nk = self.heads * c.key_dim, c.kv_heads * c.key_dim
        q = rows[:, :nq].unflatten(1, (self.heads, c.key_dim))
        k = rows[:, nq:nq + nk].unflatten(1, (c.kv_heads, c.key_dim))
        v = rows[:, nq + nk:].unflatten(1, (c.kv_heads, c.value_dim))
        if self.rotary is not None:
            q = self.rotary.apply(q, positions, out=q)
        c.append(k, v, batch, rotary=self.rotary)
        o = q.new_zeros((h.shape[0], self.heads, c.value_dim))   # attend leaves rows of no sequence as they were
        o = c.attend(q, batch, scale=self.scale, window=self.window, out=o).flatten(1)
        if out_f32 is None:
            return o @ self.wo.T
        if (self.wo.requires_grad and torch.is_grad_enabled()) or _dual(self.wo):
            return out_f32.copy_(o @ self.wo.T)   # torch has no derivative of the product below
        return torch.mm(o, self.wo.T, out_dtype=_F32, out=out_f32)

    __call__ = forward


def make_attention(n_layers, hidden, heads, kv_heads, key_dim, value_dim, pages, *, rotary=None, device="cuda", seed=0, window=0):
    """Synthetic attention halves (seeded weights, empty caches of `pages` pages)."""
    g = torch.Generator().manual_seed(seed)

    def weight(n, m):
        return (torch.randn(n, m, generator=g) * m ** -0.5).to(_BF16).to(device)

    rows = heads * key_dim + kv_heads * (key_dim + value_dim)
    return [PagedAttention(PagedKVCache(pages, kv_heads, key_dim, value_dim, device=device), weight(rows, hidden),
                           weight(hidden, heads * value_dim), heads, rotary, window=window) for _ in range(n_layers)]
