"""4-bit key/value cache: rotary positions, append and attention on the B200.

The weights' groupwise INT4 format (openquant/groupwise.py:13-61 of the
reference, which quantizes weights only) carried over to the keys and values
of a decoding model.  One layer's cache is paged:

    k_codes, v_codes    uint8 [pages, kv_heads, page_size, head_dim / 2]
    k_scales, v_scales  fp16  [pages, kv_heads, page_size, head_dim / group]

with two codes a byte (element 2i in the low nibble, two's complement) and one
scale per group of head_dim.  A scale is max|x| / 7 rounded to 8 significant
bits (through bf16), at most 9344, 1 where that is 0; a code is
clip(rint(x / scale), -7, 7).  Every cached value code * scale is exactly an
fp16 number, so attention multiplies it on the tensor cores unrounded.

A step of a serving loop, for each layer:

    batch = KVBatch(page_table, lengths)             # one new token per sequence
    q = cache.append(k, v, batch, q=q, table=table)  # rotates q and k, writes k and v
    y = cache.attention(q, batch)

Everything is asynchronous on the current CUDA stream of the tensors' GPU.
Only rotary() has a gradient: the cache is for inference, and what append, read
and attention return carries no history.  There is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math
import threading

import torch

from . import _native as nat
from .triton_int4 import _stream_handle

__all__ = ["rotary_table", "rotary", "KVBatch", "Int4KVCache", "take_device_error"]

_CODES = {torch.float32: nat.OQ_F32, torch.float16: nat.OQ_F16, torch.bfloat16: nat.OQ_BF16}
_ROTARY_INTERLEAVED, _ROTARY_INVERSE = 1, 2
_NOT_CAUSAL = 1
MAX_SEQUENCES = 2048
_KEEP_BYTES, _KEEP_BUFFERS = 32 << 20, 4  # workspaces that a KVBatch keeps


def take_device_error():
    """Reads and clears the library's device error word of the current GPU,
    after the work on it has ended: 0, or what a kernel met first -- 1 gave up
    waiting inside a kernel (its outputs are undefined), 2 for a peer GPU, 3 a
    page number, a position or a sequence's starts outside their arrays, or more
    tokens than max_tokens (what they stand for was left out)."""
    nat.require_device()
    code = ctypes.c_int32()
    nat.check(nat.load().oq_take_device_error(ctypes.byref(code)))
    return code.value


# -------------------------------------------------------------- rotary --


def _frequencies(dim, base, scaling):
    """(angle per position of each pair, factor of cos and sin), fp64."""
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    if scaling is None:
        return base ** (-i / dim), 1.0
    kind, factor = scaling.get("type"), float(scaling.get("factor", 1.0))
    if factor <= 0:
        raise ValueError("the scaling factor must be positive")
    freq = base ** (-i / dim)
    if kind == "linear":
        return freq / factor, 1.0
    if kind == "ntk":
        if dim < 4:
            raise ValueError("ntk scaling needs a rotary dimension of at least 4")
        return (base * factor ** (dim / (dim - 2))) ** (-i / dim), 1.0
    if kind not in ("parts", "smooth"):
        raise ValueError(f"unknown rotary scaling {kind!r}")
    original = float(scaling["original_positions"])
    turns = original * freq / (2 * math.pi)  # turns of each pair over the original context
    if kind == "smooth":  # linear in the turns between low and high of them
        low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
        if not high > low:
            raise ValueError("smooth scaling needs high > low")
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return freq * (keep + (1 - keep) / factor), 1.0
    # linear in the pair's index between the pairs that turn `high` and `low` times
    low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 32.0))

    def index(n):
        return dim * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base))

    # either pair may lie outside the head: the line goes through it all the same
    first, last = math.floor(index(high)), math.ceil(index(low))
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - first) / max(last - first, 1e-3)).clamp(0, 1)
    size = float(scaling.get("magnitude", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0))
    return freq * (1 - ramp) + freq / factor * ramp, size


def rotary_table(positions, rotary_dim, *, base=10000.0, scaling=None, device=None):
    """cos | sin of the angles of positions 0 .. positions - 1: fp32
    [positions, rotary_dim] (the rotary_dim / 2 cosines of a position, then its
    sines), computed in fp64 and rounded once.  Pair i of a head turns by
    position * base^(-2i / rotary_dim).

    scaling, for contexts longer than the model was trained on, is a dict:
      {"type": "linear", "factor": f}   positions divided by f
      {"type": "ntk", "factor": f}      base * f^(d / (d - 2))
      {"type": "parts", "factor": f, "original_positions": n, "low": 1, "high": 32,
       "magnitude": ...}                pairs that turn more than `high` times over n positions keep
                                        their angle, those below `low` turns have it divided by f, linear
                                        in the pair's index between (from the last whole index that
                                        turns at least `high` times to the first that turns at most `low`
                                        times, in the head or outside it); cos and sin times magnitude
                                        (0.1 ln f + 1)
      {"type": "smooth", "factor": f, "original_positions": n, "low": 1, "high": 4}
                                        the same with a passage linear in the number of turns
    """
    positions, rotary_dim = int(positions), int(rotary_dim)
    if positions < 1:
        raise ValueError("positions must be positive")
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even and at least 2")
    if base <= 0:
        raise ValueError("base must be positive")
    freq, size = _frequencies(rotary_dim, float(base), scaling)
    freq = freq.to(device if device is not None else "cuda")
    angle = torch.arange(positions, dtype=torch.float64, device=freq.device)[:, None] * freq
    return torch.cat([angle.cos() * size, angle.sin() * size], dim=1).float()


class _RotarySpec(ctypes.Structure):
    _fields_ = [("table", ctypes.c_void_p), ("rows", ctypes.c_int64), ("dim", ctypes.c_int32),
                ("flags", ctypes.c_int32)]


def _rotary_spec(table, flags, head_dim, dev):
    if (not isinstance(table, torch.Tensor) or table.dtype is not torch.float32 or table.ndim != 2
            or table.get_device() != dev or not table.is_contiguous()):
        raise ValueError("table must be a contiguous float32 (positions, rotary_dim) tensor on the operands' GPU")
    rows, dim = table.shape
    if rows < 1 or dim < 2 or dim % 2 or dim > head_dim:
        raise ValueError("the table's rotary dimension must be even, at least 2 and at most head_dim")
    return _RotarySpec(table.data_ptr(), rows, dim, flags)


def _positions(positions, tokens, dev):
    if (not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64)
            or positions.shape != (tokens,) or positions.get_device() != dev or not positions.is_contiguous()):
        raise ValueError("positions must be a contiguous int32 or int64 tensor of one position per token")
    return positions.data_ptr(), 1 if positions.dtype is torch.int64 else 0


def _heads(x, name, dtypes=(torch.float16, torch.bfloat16)):
    if not isinstance(x, torch.Tensor) or x.ndim != 3 or x.dtype not in dtypes:
        raise ValueError(f"{name} must be a 3-D (tokens, heads, head_dim) tensor of "
                         + " or ".join(str(d).replace("torch.", "") for d in dtypes))
    if not x.is_cuda:
        raise ValueError("All tensors must be on CUDA")
    tokens, heads, dim = x.shape
    if not (tokens and heads and dim):
        raise ValueError(f"{name}: dimensions must be positive")
    if x.stride(2) != 1 and dim > 1:
        raise ValueError(f"{name}: the elements of a head must be contiguous")
    return tokens, heads, dim


def _like(x):
    """A contiguous tensor like x (empty_like, the quicker call, keeps strides)."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _call(dev, fn, *args):
    """fn(*args, stream) on the tensors' GPU, its status checked."""
    if torch.cuda.current_device() == dev:
        st = fn(*args, _stream_handle(dev))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, _stream_handle(dev))
    if st:
        nat.check(st)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, table, positions, interleaved, inverse):
        ctx.save_for_backward(table, positions)
        ctx.interleaved, ctx.inverse = interleaved, inverse
        return rotary(x, table, positions, interleaved=interleaved, inverse=inverse)

    @staticmethod
    def backward(ctx, g):
        table, positions = ctx.saved_tensors
        if g.stride(2) != 1:
            g = g.contiguous()
        return rotary(g, table, positions, interleaved=ctx.interleaved, inverse=not ctx.inverse), None, None, None, None


def rotary(x, table, positions, *, interleaved=False, inverse=False, out=None):
    """Rotary positions: x [tokens, heads, head_dim] (fp32, fp16 or bf16 on a
    GPU; tokens and heads may be strided) with every token's heads turned by
    the token's position, in fp32 and rounded once to x's dtype.

    table (rotary_table) has one row per position; its width, the rotary
    dimension, may be less than head_dim (the rest of a head is copied).
    Pairs are (i, i + rotary_dim / 2), or (2i, 2i + 1) with interleaved=True:
    (a, b) becomes (a cos - b sin, b cos + a sin).  inverse=True turns by the
    negative angle: the transpose of the rotation, which takes the gradient of
    y to that of x (and y back to x, where the table's magnitude is 1).  out may
    be x itself.  Where x needs a gradient the call is recorded by autograd,
    its gradient being the same kernel with the other sign; out cannot be given
    then, and the table has no gradient.
    positions (int32 or int64 [tokens]) outside the table leave their tokens'
    output unwritten and set the device error (take_device_error) to 3.
    """
    tokens, heads, dim = _heads(x, "x", (torch.float32, torch.float16, torch.bfloat16))
    if dim % 8 or dim > 256:
        raise ValueError("head_dim must be a multiple of 8 up to 256")
    dev = x.get_device()
    spec = _rotary_spec(table, (_ROTARY_INTERLEAVED if interleaved else 0) | (_ROTARY_INVERSE if inverse else 0), dim,
                        dev)
    pos, wide = _positions(positions, tokens, dev)
    if (x.requires_grad or table.requires_grad) and torch.is_grad_enabled():
        if table.requires_grad:
            raise ValueError("the table has no gradient")
        if out is not None:
            raise ValueError("out cannot be given where x needs a gradient")
        return _Rotary.apply(x, table, positions, bool(interleaved), bool(inverse))
    if out is None:
        out = _like(x)
    elif (out.shape != x.shape or out.dtype is not x.dtype or out.get_device() != dev
          or (out.stride(2) != 1 and dim > 1)):
        raise ValueError("out must be like x, with contiguous heads")
    nat.require_device()
    xs, ys = x.stride(), out.stride()
    _call(dev, nat.load().oq_rotary, x.data_ptr(), out.data_ptr(), _CODES[x.dtype], tokens, heads, dim, xs[0], xs[1],
          ys[0], ys[1], ctypes.byref(spec), pos, wide)
    return out


# --------------------------------------------------------------- cache --


class _Batch(ctypes.Structure):
    _fields_ = [("page_table", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("starts", ctypes.c_void_p),
                ("sequences", ctypes.c_int32), ("max_pages", ctypes.c_int32), ("max_tokens", ctypes.c_int32)]


class _Cache(ctypes.Structure):
    _fields_ = [("k_codes", ctypes.c_void_p), ("k_scales", ctypes.c_void_p), ("v_codes", ctypes.c_void_p),
                ("v_scales", ctypes.c_void_p), ("pages", ctypes.c_int64), ("page_size", ctypes.c_int32),
                ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("group_size", ctypes.c_int32)]


class KVBatch:
    """The sequences of one step, checked once and used by every layer.

    page_table int32 [sequences, max_pages]: the page of a sequence's tokens
    j // page_size.  lengths int32 [sequences]: its tokens in the cache with
    the step's own, which are its last ones.  starts int32 [sequences + 1]
    (starts[0] = 0): sequence b's tokens of the step's arrays are
    [starts[b], starts[b + 1]); None: one token per sequence.  Tokens from
    starts[-1] on are padding.  max_tokens: an upper bound of the tokens per
    sequence, known on the host (needed with starts); attention leaves out a
    sequence with more (rows of 0, log-sum -inf, device error 3).

    The tensors are read by the kernels, so their contents may change between
    steps (a captured CUDA graph replays with the new ones).  A page number or
    position outside its array is not followed, and a sequence whose starts
    are not in order within the step's arrays is left out (nothing is written,
    rows of 0): the device error (take_device_error) becomes 3.
    """

    def __init__(self, page_table, lengths, starts=None, *, max_tokens=None):
        for t, name in ((page_table, "page_table"), (lengths, "lengths"), (starts, "starts")):
            if t is None and name == "starts":
                continue
            if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32:
                raise ValueError(f"{name} must be an int32 tensor")
            if not t.is_cuda:
                raise ValueError("All tensors must be on CUDA")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        if page_table.ndim != 2 or min(page_table.shape) < 1:
            raise ValueError("page_table must be a nonempty 2-D (sequences, max_pages) tensor")
        n = int(page_table.shape[0])
        if n > MAX_SEQUENCES:
            raise ValueError(f"a batch has at most {MAX_SEQUENCES} sequences")
        if lengths.shape != (n,):
            raise ValueError("lengths must have one element per sequence")
        if starts is not None and starts.shape != (n + 1,):
            raise ValueError("starts must have one element more than there are sequences")
        dev = page_table.get_device()
        if lengths.get_device() != dev or (starts is not None and starts.get_device() != dev):
            raise ValueError("All tensors must use the same GPU")
        if max_tokens is None:
            if starts is not None:
                raise ValueError("max_tokens is needed with starts")
            max_tokens = 1
        max_tokens = int(max_tokens)
        if max_tokens < 1 or (starts is None and max_tokens != 1):
            raise ValueError("max_tokens must be positive, and 1 without starts")
        if max_tokens >= 1 << 31:
            raise ValueError("max_tokens must be below 2^31")
        self.page_table, self.lengths, self.starts = page_table, lengths, starts
        self.sequences, self.max_tokens = n, max_tokens
        self._dev = dev
        self._c = _Batch(page_table.data_ptr(), lengths.data_ptr(), starts.data_ptr() if starts is not None else None,
                         n, int(page_table.shape[1]), max_tokens)
        self._ref = ctypes.byref(self._c)
        self._ws = {}  # (cache shape, q_heads, tokens) -> workspace bytes
        self._buffers = {}  # (stream, host thread) -> workspace

    def _workspace(self, nbytes, device):
        """nbytes of scratch memory for a call on the current stream.  A call is
        several kernels that hand results on through it: one buffer per stream
        and host thread, as only the launches of one thread on one stream are
        sure to follow each other call by call (two threads on the stream that
        they share by default may launch theirs in turn).  A captured call has
        its own from the graph's pool, and large ones are not kept."""
        if nbytes > _KEEP_BYTES or torch.cuda.is_current_stream_capturing():
            return torch.empty(nbytes, dtype=torch.uint8, device=device)
        key = (_stream_handle(self._dev), threading.get_ident())
        buf = self._buffers.get(key)
        if buf is None or buf.numel() < nbytes:
            if len(self._buffers) >= _KEEP_BUFFERS:
                self._buffers.clear()
            buf = self._buffers[key] = torch.empty(nbytes, dtype=torch.uint8, device=device)
        return buf


class Int4KVCache:
    """One layer's paged 4-bit key/value cache (see the module's docstring for
    the arrays).  The object holds the four tensors it is given; allocate()
    makes them.  head_dim is 64 or 128, the group 32, 64 or 128 (at most
    head_dim), page_size a multiple of 16.

    A key or value that is NaN or infinite makes the keys of its token and
    head read as NaN: every query that sees the token gets NaN, no other does.
    """

    def __init__(self, k_codes, k_scales, v_codes, v_scales):
        for t, name in ((k_codes, "k_codes"), (v_codes, "v_codes")):
            if not isinstance(t, torch.Tensor) or t.dtype is not torch.uint8 or t.ndim != 4:
                raise ValueError(f"{name} must be a 4-D uint8 tensor (pages, kv_heads, page_size, head_dim / 2)")
        for t, name in ((k_scales, "k_scales"), (v_scales, "v_scales")):
            if not isinstance(t, torch.Tensor) or t.dtype is not torch.float16 or t.ndim != 4:
                raise ValueError(f"{name} must be a 4-D float16 tensor (pages, kv_heads, page_size, groups)")
        every = (k_codes, k_scales, v_codes, v_scales)
        if not all(t.is_cuda for t in every):
            raise ValueError("All tensors must be on CUDA")
        if not all(t.is_contiguous() for t in every):
            raise ValueError("The cache's tensors must be contiguous")
        if k_codes.shape != v_codes.shape or k_scales.shape != v_scales.shape:
            raise ValueError("keys and values must have the same shapes")
        pages, kv_heads, page_size, half = (int(v) for v in k_codes.shape)
        groups = int(k_scales.shape[3])
        if tuple(k_scales.shape[:3]) != (pages, kv_heads, page_size) or min(k_codes.shape) < 1 or groups < 1:
            raise ValueError("scales must have one row per row of codes")
        head_dim = 2 * half
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if head_dim % groups or head_dim // groups not in (32, 64, 128):
            raise ValueError("Group size must be 32, 64 or 128")
        if page_size % 16:
            raise ValueError("page_size must be a positive multiple of 16")
        if len({t.get_device() for t in every}) != 1:
            raise ValueError("All tensors must use the same GPU")
        if any(t.data_ptr() % 16 for t in every):
            raise ValueError("The cache's tensors must be 16-byte aligned")
        nat.require_device()
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = every
        self.pages, self.page_size, self.kv_heads = pages, page_size, kv_heads
        self.head_dim, self.group_size = head_dim, head_dim // groups
        self._dev = k_codes.get_device()
        self._device = k_codes.device
        self._lib = nat.load()
        self._c = _Cache(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(), pages,
                         page_size, kv_heads, head_dim, self.group_size)
        self._ref = ctypes.byref(self._c)
        self._key = (kv_heads, head_dim, page_size)

    @classmethod
    def allocate(cls, pages, page_size, kv_heads, head_dim, group_size=32, *, device="cuda"):
        """A cache of zeros: pages * page_size tokens of kv_heads heads."""
        pages, page_size, kv_heads = int(pages), int(page_size), int(kv_heads)
        if pages < 1 or kv_heads < 1 or page_size < 1:
            raise ValueError("Cache dimensions must be positive")
        if head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if group_size not in (32, 64, 128) or group_size > head_dim:
            raise ValueError("Group size must be 32, 64 or 128, at most head_dim")
        if page_size % 16:
            raise ValueError("page_size must be a positive multiple of 16")

        def codes():
            return torch.zeros((pages, kv_heads, page_size, head_dim // 2), dtype=torch.uint8, device=device)

        def scales():
            return torch.zeros((pages, kv_heads, page_size, head_dim // group_size), dtype=torch.float16,
                               device=device)

        return cls(codes(), scales(), codes(), scales())

    def _check_batch(self, batch, dev):
        if not isinstance(batch, KVBatch):
            raise ValueError("batch must be a KVBatch")
        if batch._dev != self._dev or dev != self._dev:
            raise ValueError("All tensors must use the same GPU")

    def append(self, k, v, batch, *, q=None, table=None, positions=None, interleaved=False, q_out=None):
        """Writes the step's keys and values k, v [tokens, kv_heads, head_dim]
        (fp16 or bf16, tokens and heads may be strided) into the batch's pages,
        at the ends of its sequences, as 4-bit codes and scales.  With a rotary
        table, keys are rotated first (in fp32, without another rounding) by
        their place in the sequence, or by `positions` ([tokens], int32 or
        int64) where given; q [tokens, heads, head_dim] is rotated likewise and
        returned in q's dtype (q_out, which may be q, takes it; None without
        q).  A token whose position is outside the table is not written,
        neither to the cache nor to q's output.  One kernel."""
        tokens, heads, dim = _heads(k, "k")
        if heads != self.kv_heads or dim != self.head_dim:
            raise ValueError("k must have the cache's kv_heads and head_dim")
        if not isinstance(v, torch.Tensor) or v.shape != k.shape or v.dtype is not k.dtype:
            raise ValueError("v must have k's shape and dtype")
        vs = v.stride()
        if vs[2] != 1:
            raise ValueError("v: the elements of a head must be contiguous")
        dev = k.get_device()
        self._check_batch(batch, dev)
        if v.get_device() != dev:
            raise ValueError("All tensors must use the same GPU")
        if table is None and (q is not None or positions is not None):
            raise ValueError("q and positions need a rotary table")
        if q is None:
            if q_out is not None:
                raise ValueError("q_out needs q")
            qa = (None, None, 0, 0, 0, 0, 0)
        else:
            qt, qh, qd = _heads(q, "q")
            if qt != tokens or qd != dim or q.dtype is not k.dtype or q.get_device() != dev:
                raise ValueError("q must have k's tokens, head_dim, dtype and GPU")
            if q_out is None:
                q_out = _like(q)
            elif (q_out.shape != q.shape or q_out.dtype is not q.dtype or q_out.get_device() != dev
                  or q_out.stride(2) != 1):
                raise ValueError("q_out must be like q, with contiguous heads")
            qs, os = q.stride(), q_out.stride()
            qa = (q.data_ptr(), q_out.data_ptr(), qh, qs[0], qs[1], os[0], os[1])
        spec, pos, wide = None, None, 0
        if table is not None:
            spec = ctypes.byref(_rotary_spec(table, _ROTARY_INTERLEAVED if interleaved else 0, dim, dev))
            if positions is not None:
                pos, wide = _positions(positions, tokens, dev)
        ks = k.stride()
        _call(dev, self._lib.oq_kv4_append, self._ref, batch._ref, *qa, k.data_ptr(), ks[0], ks[1], v.data_ptr(),
              vs[0], vs[1], _CODES[k.dtype], tokens, spec, pos, wide)
        return q_out

    def read(self, batch, tokens, *, dtype=torch.float16):
        """What the cache holds of the batch's own tokens (`tokens` of them):
        k, v [tokens, kv_heads, head_dim] = code * scale, exact in fp16 and
        fp32.  A batch whose starts cover whole sequences reads those."""
        tokens = int(tokens)
        if tokens < 1:
            raise ValueError("tokens must be positive")
        if dtype not in _CODES:
            raise ValueError("dtype must be torch.float16, torch.bfloat16 or torch.float32")
        self._check_batch(batch, self._dev)
        k, v = torch.empty((2, tokens, self.kv_heads, self.head_dim), dtype=dtype, device=self._device).unbind(0)
        _call(self._dev, self._lib.oq_kv4_read, self._ref, batch._ref, k.data_ptr(), v.data_ptr(), _CODES[dtype],
              tokens)
        return k, v

    def attention(self, q, batch, *, scale=None, window=0, causal=True, out=None, return_log_sum=False):
        """softmax(scale * q . K^T + mask) . V over the batch's sequences.

        q [tokens, heads, head_dim] (fp16 or bf16, tokens and heads may be
        strided; rotated already) are the step's queries, heads a multiple of
        kv_heads: query head i uses key head i // (heads / kv_heads).  scale is
        1 / sqrt(head_dim) by default.  A query at position p of its sequence
        sees positions <= p (causal=False: all), and with window > 0 only those
        > p - window.  Returns [tokens, heads, head_dim] in q's dtype (out, a
        contiguous tensor, where given), and with return_log_sum also fp32
        [tokens, heads] log sum exp(scale q.k).  A row that sees nothing is 0
        with log-sum -inf, and so are padding tokens."""
        tokens, heads, dim = _heads(q, "q")
        if dim != self.head_dim:
            raise ValueError("q must have the cache's head_dim")
        if heads % self.kv_heads:
            raise ValueError("q's heads must be a multiple of kv_heads")
        dev = q.get_device()
        self._check_batch(batch, dev)
        window = int(window or 0)
        if window < 0:
            raise ValueError("window must not be negative")
        window = min(window, 1 << 31)  # no limit
        scale = dim ** -0.5 if scale is None else float(scale)
        if not math.isfinite(scale):
            raise ValueError("scale must be finite")
        if out is None:
            out = _like(q)
        elif (out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != dev
              or not out.is_contiguous()):
            raise ValueError("out must be a contiguous tensor like q")
        log_sum = torch.empty((tokens, heads), dtype=torch.float32, device=self._device) if return_log_sum else None
        key = (*self._key, heads, tokens)
        ws_bytes = batch._ws.get(key)
        if ws_bytes is None:
            with torch.cuda.device(dev):
                ws_bytes = self._lib.oq_kv4_attention_workspace_bytes(self._ref, batch._ref, heads, tokens)
            if ws_bytes <= 0:
                raise RuntimeError(nat.last_error() or "kv4_attention: no workspace size")
            batch._ws[key] = ws_bytes
        if torch.cuda.current_device() != dev:  # the workspace is the current stream's
            with torch.cuda.device(dev):
                ws = batch._workspace(ws_bytes, self._device)
        else:
            ws = batch._workspace(ws_bytes, self._device)
        qs = q.stride()
        _call(dev, self._lib.oq_kv4_attention, self._ref, batch._ref, q.data_ptr(), _CODES[q.dtype], heads, qs[0],
              qs[1], out.data_ptr(), log_sum.data_ptr() if return_log_sum else None, tokens, scale, window,
              0 if causal else _NOT_CAUSAL, ws.data_ptr(), ws_bytes)
        return (out, log_sum) if return_log_sum else out
