"""Token operators on MI355X: the layers of an attention block over the tokens of camera frames.

* ``Linear`` -- a matrix product with bias, activation and residual in its epilogue (bf16, f32 or e4m3 weights);
* ``QKNorm`` with ``Rotary`` -- the norms of queries and keys for each head and the rotation by the token's position
  on one or more axes (time, height, width) in one pass, into a ``TokenCache`` where a stream keeps one;
* ``attend`` -- attention by frames with a sliding window and first tokens that stay visible (sinks).

Each call is one launch or two of ``libva355.so`` (``va_tok_linear`` / ``va_tok_qk`` / ``va_tok_attn`` in va355.h) on
the current stream of the tensors' device, or on ``stream``; it does not synchronise, keeps nothing between calls and may
be captured into a graph.  Results are the same from call to call, bit by bit.  With ``stream``, what the call allocates
belongs to that stream, its inputs are recorded on it, and the caller orders it against the work that made them.

The operators are forward only, as every layer of this package: a tensor that requires a gradient is refused while
gradients are recorded (weights are copied when a layer is made, and may require one).
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import struct

import torch

from . import _lib
from .seg import VA_DTYPE_BF16, VA_DTYPE_F32, split3_bf16

VOIDP, I32, I64, F32 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
ACTS = {None: 0, "none": 0, "silu": 1, "gelu": 2, "gelu_tanh": 3, "relu": 4}
LAYOUTS = {"half": 0, "pairs": 1}
DTYPES = {torch.bfloat16: VA_DTYPE_BF16, torch.float32: VA_DTYPE_F32}
I32_MAX = 2 ** 31 - 1


class LinearArgs(ctypes.Structure):  # va_tok_linear_args
    _fields_ = [(n, VOIDP) for n in ("x", "w", "wscale", "bias", "res", "y")] + \
               [(n, I64) for n in ("ldx", "ldr", "ldy")] + \
               [(n, I32) for n in ("M", "N", "K", "Npad", "Kpad", "dtype", "w8", "act", "out_f32", "pad")]


class QKArgs(ctypes.Structure):  # va_tok_qk_args
    _fields_ = [(n, VOIDP) for n in ("q", "k", "v", "q_out", "k_out", "v_out")] + \
               [(f"{t}_{d}", I64) for t in ("q", "k", "v", "qo", "ko", "vo") for d in ("sb", "ss", "sh")] + \
               [("q_weight", VOIDP), ("k_weight", VOIDP), ("eps", F32), ("rot", I32), ("turns", VOIDP), ("axis", VOIDP),
                ("pos", VOIDP), ("pos_sb", I64), ("pos_ss", I64), ("q_len", VOIDP), ("kv_len", VOIDP)] + \
               [(n, I32) for n in ("B", "S", "Hq", "Hk", "D", "Dv", "axes", "layout", "slots", "sinks", "dtype", "pad")]


class AttnArgs(ctypes.Structure):  # va_tok_attn_args
    _fields_ = [(n, VOIDP) for n in ("q", "k", "v", "o")] + \
               [(f"{t}_{d}", I64) for t in ("q", "k", "v", "o") for d in ("sb", "ss", "sh")] + \
               [("q_len", VOIDP), ("kv_len", VOIDP), ("scale", F32)] + \
               [(n, I32) for n in ("B", "S", "Hq", "Hk", "D", "Dv", "slots", "frame", "window", "sinks", "dtype")] + \
               [("ws", VOIDP), ("ws_bytes", I64)]


# the same layouts for a call's own use: one pack() of plain numbers is a fraction of a ctypes structure's fields, and
# small calls are bound by the host
LINEAR_PACK = struct.Struct("@6P3q10i")
QK_PACK = struct.Struct("@6P18q2Pfi3P2q2P12i")
ATTN_PACK = struct.Struct("@4P12q2Pf11iPq")
assert (LINEAR_PACK.size, QK_PACK.size, ATTN_PACK.size) == tuple(ctypes.sizeof(t) for t in (LinearArgs, QKArgs, AttnArgs))


# ------------------------------------------------------------------ what every call checks
def _need(ok: bool, what: str) -> None:
    if not ok:
        raise _lib.VaError(what)


def _on(t: torch.Tensor, dev: torch.device, dtype, name: str) -> None:
    if t.device != dev:
        raise _lib.VaError(f"{name} is on {t.device}, not on {dev}")
    if t.dtype != dtype:
        raise _lib.VaError(f"{name} is {t.dtype}, not {dtype}")
    if t.requires_grad:
        _no_grad(name)


def _no_grad(name: str) -> None:
    """Refuses a tensor that requires a gradient where one would be recorded: the result would be cut off from it."""
    if torch.is_grad_enabled():
        raise _lib.VaError(f"{name} requires a gradient, and the token operators are forward only: detach() it, or call under "
                           "torch.no_grad()")


def _gpu(device) -> torch.device:
    """The GPU that a layer is made on (None: the current one)."""
    d = torch.device("cuda" if device is None else device)
    _need(d.type == "cuda", f"device {d}: the token operators run on the GPU")
    return d if d.index is not None else torch.device("cuda", torch.cuda.current_device())


def _floats(t: torch.Tensor | None, dev: torch.device) -> torch.Tensor | None:
    """A layer's own copy of a vector, as its weights are one: the caller's may change later."""
    return None if t is None else t.detach().to(dev, torch.float32, copy=True, memory_format=torch.contiguous_format)


def _range(t: torch.Tensor) -> tuple[int, int]:
    """The bytes between a tensor's first and last element (0, 0: it has none)."""
    if t.is_contiguous():
        at = t.data_ptr()
        return at, at + t.numel() * t.element_size()
    if t.numel() == 0:
        return 0, 0
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _interleaved(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether two tensors of one type repeat with a common period and keep to parts of it that do not meet (queries and
    keys as views of one product's output)."""
    if x.dtype != y.dtype or x.dim() != y.dim() or (y.data_ptr() - x.data_ptr()) % x.element_size():
        return False
    at = (y.data_ptr() - x.data_ptr()) // x.element_size()
    dims = [(m, a, n, b) for m, a, n, b in zip(x.shape, x.stride(), y.shape, y.stride())]
    for p in {a for m, a, n, b in dims if a == b and a > 0}:
        outer = [d for d in dims if max(d[1] if d[0] > 1 else 0, d[3] if d[2] > 1 else 0) >= p]
        if any(a != b or a % p for m, a, n, b in outer):
            continue
        inner = [d for d in dims if d not in outer]
        lx, ly = (1 + sum((d[i] - 1) * d[i + 1] for d in inner) for i in (0, 2))
        if at % p >= lx and at % p + ly <= p:
            return True
    return False


def _plain(t: torch.Tensor, item: int) -> tuple:
    """A 4-d tensor as (address, its strides, the end of its bytes)."""
    at = t.data_ptr()
    a, b, c, d = t.stride()
    n, m, h, w = t.shape
    return at, a, b, c, d, at + ((n - 1) * a + (m - 1) * b + (h - 1) * c + (w - 1) * d + 1) * item


def _meet(x: tuple[int, int], y: tuple[int, int]) -> bool:
    return x[0] < y[1] and y[0] < x[1]


def _apart(out: torch.Tensor, t: torch.Tensor | None, name: str, same_ok: bool = False) -> None:
    """Refuses an output that overlaps an input (same_ok: unless it is that very tensor)."""
    if t is None:
        return
    if _meet(_range(out), _range(t)) and not (same_ok and out.data_ptr() == t.data_ptr() and out.shape == t.shape and
                                out.stride() == t.stride() and out.dtype == t.dtype) \
            and not _interleaved(out, t):
        raise _lib.VaError(f"the output overlaps {name}")


def _own_elements(out: torch.Tensor) -> None:
    """Refuses an output whose elements share memory (an expanded tensor)."""
    if out.is_contiguous():
        return
    at = 1
    for s, n in sorted((s, n) for n, s in zip(out.shape, out.stride()) if n > 1):
        _need(s >= at, "the output's elements overlap")
        at = s * n


def _fixed(name: str) -> property:
    """A tensor whose address a call takes from the object: it is read, not replaced (its values may change)."""
    return property(lambda self: self.__dict__["_" + name])


_raw_stream, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _elsewhere(dev: torch.device, stream, inputs, go):
    """go() on a device that is not the current one, or on a stream of the caller's: what it allocates belongs to that
    stream, and its inputs are recorded on it."""
    if dev.type != "cuda":
        raise _lib.VaError(f"the token operators need tensors on the GPU, not on {dev}")
    with contextlib.ExitStack() as scope:
        scope.enter_context(torch.cuda.device(dev))
        if stream is not None:
            _lib.stream_ptr(stream, dev)  # refuses a stream of another device
            scope.enter_context(torch.cuda.stream(stream))
            for t in inputs:
                if t is not None:
                    t.record_stream(stream)
        return go()


def _here(dev: torch.device, stream) -> bool:
    return stream is None and dev.type == "cuda" and dev.index == _device()


# ------------------------------------------------------------------ matrix product
def _blocks(w: torch.Tensor) -> torch.Tensor:
    """[N, K] (multiples of 32; bf16 or bytes) in the packed order of va_tok_linear_args.w: [K / 32, N / 32, 32, 32]."""
    N, K = w.shape
    r = torch.arange(32, device=w.device)
    ch = 16 * (r // 4 % 2) + 4 * (r // 8) + r % 4
    turn = r // (4 if w.element_size() == 2 else 8) % 4
    col = 8 * (torch.arange(4, device=w.device) ^ turn[:, None])[:, :, None] + torch.arange(8, device=w.device)
    b = w.view(N // 32, 32, K // 32, 32).permute(2, 0, 1, 3)
    return b[:, :, ch].gather(3, col.reshape(32, 32).expand(b.shape)).contiguous()


def _terms(w: torch.Tensor) -> torch.Tensor:
    """[N, K] float -> its bf16 terms h, m, l [3, N, K], of any value (va355.h va_tok_linear_args.w)."""
    t = split3_bf16(w).permute(2, 0, 1, 3).reshape(3, *w.shape)
    far = w.abs() >= float.fromhex("0x1.ffp127")
    if not far.any():
        return t
    (h, m, l), inf = t, w.isinf()
    h = torch.where(far, torch.where(inf, 1.0, torch.finfo(torch.bfloat16).max).copysign(w).to(h.dtype), h)
    r = torch.where(far, w - h.float(), 0.0)
    m = torch.where(inf, 0.0, torch.where(far, r.to(h.dtype), m))
    l = torch.where(far, torch.where(inf, w, r - m.float()).to(h.dtype), l)
    return torch.stack([h, m, l])


class Linear:
    """y = act(x w^T + bias) + residual, the weights packed once.

    weight: [N, K].  dtype "bf16" (bf16 tensors), "f32" (float tensors; every product as six exact bf16 term products,
    float sums) or "w8a16" (bf16 tensors, e4m3 weight bytes with one float scale per row: quantised here as the
    convolutions' are, or given as float8_e4m3fn values with ``scale`` [N]).  bias: [N].  act: None, "silu", "gelu",
    "gelu_tanh" or "relu"."""

    w, wscale, bias = _fixed("w"), _fixed("wscale"), _fixed("bias")

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, act: str | None = None,
                 dtype: str = "bf16", scale: torch.Tensor | None = None, device=None):
        _need(dtype in ("bf16", "f32", "w8a16"), f"dtype {dtype!r}: bf16, f32 or w8a16")
        _need(act in ACTS, f"act {act!r}: {', '.join(str(a) for a in ACTS)}")
        _need(weight.dim() == 2 and weight.shape[0] > 0 and weight.shape[1] > 0, f"weight {tuple(weight.shape)}: [N, K]")
        N, K = weight.shape
        _need(max(N, K) <= I32_MAX - 64, "weight: a side beyond 32 bits")
        _need(bias is None or bias.shape == (N,), "bias: [N]")
        _need(scale is None or (dtype == "w8a16" and scale.shape == (N,) and weight.dtype == torch.float8_e4m3fn),
              "scale: [N], with float8_e4m3fn weights and dtype w8a16 only")
        _need(scale is not None or weight.dtype != torch.float8_e4m3fn, "float8_e4m3fn weights need their scale")
        _lib.require_gpu()
        self.device = _gpu(weight.device if device is None and weight.device.type == "cuda" else device)
        self.lib = _lib.load()
        self.N, self.K, self.dtype = N, K, dtype
        self.tdtype = torch.float32 if dtype == "f32" else torch.bfloat16
        Np, Kp = -(-N // 64) * 64, -(-K // 64) * 64

        def padded(t):
            p = torch.zeros(Np, Kp, dtype=t.dtype, device=self.device)
            p[:N, :K] = t
            return p

        w, self._wscale = weight.detach().to(self.device), None
        if dtype == "w8a16":
            if scale is None:
                from .seg import F8_MAX
                w = w.float()
                amax = w.abs().amax(1)
                scale = torch.where(amax > 0, amax / F8_MAX, torch.ones_like(amax))
                w = (w / scale[:, None]).clamp(-F8_MAX, F8_MAX).to(torch.float8_e4m3fn)
            self._wscale = torch.ones(Np, dtype=torch.float32, device=self.device)
            self._wscale[:N] = scale.detach().to(self.device, torch.float32)
            self._w = _blocks(padded(w.view(torch.uint8)))
        elif dtype == "f32":
            self._w = torch.stack([_blocks(t) for t in _terms(padded(w.float()))])
        else:
            self._w = _blocks(padded(w.to(torch.bfloat16)))
        self._bias = _floats(bias, self.device)
        self._ptrs = (self._w.data_ptr(), self._wscale.data_ptr() if self._wscale is not None else 0,
                      self._bias.data_ptr() if bias is not None else 0)
        self._ints = (N, K, Np, Kp, VA_DTYPE_F32 if dtype == "f32" else VA_DTYPE_BF16, int(dtype == "w8a16"), ACTS[act])

    def args(self, x: torch.Tensor, out: torch.Tensor, residual: torch.Tensor | None = None) -> LinearArgs:
        """The va_tok_linear_args of a call on [M, K] rows (for an op list: VA_OP_TOK_LINEAR); they point into these
        tensors and this layer's weights, which the caller keeps."""
        _need(x.dim() == 2 and x.shape[1] == self.K and x.shape[0] <= I32_MAX, f"x {tuple(x.shape)}: [M, {self.K}]")
        _on(x, self.device, self.tdtype, "x")
        want = (x.shape[0], self.N)
        if residual is not None:
            _on(residual, self.device, self.tdtype, "residual")
            _need(residual.shape == want, f"residual {tuple(residual.shape)}: {want}")
        for t, n, what in ((x, self.K, "x"), (residual, self.N, "residual")):
            _need(t is None or self._rows(t, n) is t, f"{what}: rows apart from each other, of contiguous values")
        out = self._given(out, want, x, residual)
        return LinearArgs.from_buffer_copy(self._pack(x, out, residual))

    def _pack(self, x, out, residual) -> bytes:
        M, N = x.shape[0], self.N
        one = M <= 1  # a single row's stride says nothing
        return LINEAR_PACK.pack(x.data_ptr(), *self._ptrs, 0 if residual is None else residual.data_ptr(), out.data_ptr(),
                                self.K if one else x.stride(0), N if one or residual is None else residual.stride(0),
                                N if one else out.stride(0), M, *self._ints, out.dtype != self.tdtype, 0)

    def __call__(self, x: torch.Tensor, residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 stream=None) -> torch.Tensor:
        """x [..., K] -> [..., N].  residual [..., N] is added after the activation.  out: bf16 or (for the bf16 forms)
        float; it may be the residual itself, and must not overlap x."""
        _on(x, self.device, self.tdtype, "x")
        if not _here(self.device, stream):
            return _elsewhere(self.device, stream, (x, residual, out, self.w, self.wscale, self.bias), lambda: self(x, residual, out))
        shape = x.shape
        if len(shape) == 0 or shape[-1] != self.K:
            raise _lib.VaError(f"x {tuple(shape)}: [..., {self.K}]")
        want = (*shape[:-1], self.N)
        x2 = self._rows(x, self.K)
        if x2.shape[0] > I32_MAX:
            raise _lib.VaError("more rows than 32 bits count")
        r2 = None
        if residual is not None:
            _on(residual, self.device, self.tdtype, "residual")
            if residual.shape != want:
                raise _lib.VaError(f"residual {tuple(residual.shape)}: {want}")
            r2 = self._rows(residual, self.N)
        if out is None:
            out = x.new_empty(want)
            o2 = out if len(want) == 2 else out.view(-1, self.N) if x2.shape[0] else out
        else:
            o2 = self._given(out, want, x, r2)
        if x2.shape[0]:
            rc = self.lib.va_tok_linear(_raw_stream(self.device.index), self._pack(x2, o2, r2))
            if rc:
                _lib.check(rc, "va_tok_linear")
        return out

    def _given(self, out, want, x, r2):
        """The caller's output as rows."""
        _need(out.dtype in (self.tdtype, torch.float32), f"out is {out.dtype}")
        _on(out, self.device, out.dtype, "out")
        _need(out.shape == want, f"out {tuple(out.shape)}: {want}")
        _own_elements(out)
        try:
            o2 = out.view(-1, self.N) if out.numel() else out.reshape(0, self.N)
        except RuntimeError:
            o2 = None
        _need(o2 is not None and (self.N == 1 or o2.numel() == 0 or o2.stride(1) == 1),
              "out: rows of a common stride with contiguous values")
        _apart(o2, x, "x")
        _apart(o2, r2, "the residual", same_ok=True)
        return o2

    @staticmethod
    def _rows(x: torch.Tensor, n: int) -> torch.Tensor:
        """x as rows of n contiguous values (a copy only where its strides are none)."""
        x = x.reshape(-1, n) if x.dim() != 2 else x
        return x if (x.stride(1) == 1 or n == 1) and (x.shape[0] <= 1 or x.stride(0) >= n) else x.contiguous()


# ------------------------------------------------------------------ norms and rotation
class Rotary:
    """Rotation of the first ``dim`` values of each head by the token's position.

    sections: rotated pairs of each axis, in the order of the frequencies (their sum is dim / 2; one axis by default).
    Pair f turns by base^(-2 f / dim) radians per position (freqs "shared"), or by base^(-f' / n) with f' its place among
    the n pairs of its axis (freqs "axis").  layout "half": pair f is values f and f + dim / 2; "pairs": 2 f and
    2 f + 1."""

    turns, axis = _fixed("turns"), _fixed("axis")

    def __init__(self, dim: int, sections=None, base: float = 10000.0, layout: str = "half", freqs: str = "shared",
                 device=None):
        _need(dim > 0 and dim % 2 == 0, f"dim {dim}: even")
        sections = [dim // 2] if sections is None else [int(n) for n in sections]
        _need(all(n >= 0 for n in sections) and sum(sections) == dim // 2, f"sections {sections}: sum {dim // 2}")
        _need(layout in LAYOUTS, f"layout {layout!r}: half or pairs")
        _need(freqs in ("shared", "axis"), f"freqs {freqs!r}: shared or axis")
        _need(base > 0, f"base {base}: positive")
        _lib.require_gpu()
        if freqs == "shared":
            e = [2 * f / dim for f in range(dim // 2)]
        else:
            e = [f / n for n in sections for f in range(n)]
        self.dim, self.sections, self.axes, self.layout = dim, sections, len(sections), layout
        self.device = _gpu(device)
        self._turns = torch.tensor([base ** -v / (2 * math.pi) for v in e], dtype=torch.float64, device=self.device)
        self._axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], dtype=torch.int32,
                                  device=self.device)


class TokenCache:
    """Keys and values of the last tokens of B streams, and of their first ``sinks`` tokens.

    k [B, slots, heads, D], v [B, slots, heads, Dv], len [B] (int32, on the device): tokens seen so far.  Position p is
    kept in slot p while p < slots; later ones take the slots behind the sinks in turn.  (attend reads heads of multiples of
    8 up to 128 values; QKNorm fills others too.)"""

    k, v, sinks, len = _fixed("k"), _fixed("v"), _fixed("sinks"), _fixed("len")

    def __init__(self, B: int, slots: int, heads: int, head_dim: int, v_dim: int | None = None, sinks: int = 0,
                 dtype: str = "bf16", device=None):
        _need(dtype in ("bf16", "f32"), f"dtype {dtype!r}: bf16 or f32")
        _need(min(B, slots, heads, head_dim) > 0, "B, slots, heads and head_dim are positive")
        _lib.require_gpu()
        t, dev = torch.float32 if dtype == "f32" else torch.bfloat16, _gpu(device)
        self._set(torch.zeros(B, slots, heads, head_dim, dtype=t, device=dev),
                  torch.zeros(B, slots, heads, v_dim or head_dim, dtype=t, device=dev), sinks,
                  torch.zeros(B, dtype=torch.int32, device=dev))

    def _set(self, k, v, sinks, length):
        _need(k.dim() == 4 and v.dim() == 4 and k.shape[:3] == v.shape[:3] and k.dtype == v.dtype and k.device == v.device,
              "k [B, slots, heads, D] and v [B, slots, heads, Dv] of one type")
        _need(0 <= sinks < k.shape[1], f"sinks {sinks}: fewer than the {k.shape[1]} slots")
        _on(length, k.device, torch.int32, "length")
        _need(length.shape == (k.shape[0],) and length.is_contiguous(), "length: [B]")
        _need(k.stride(3) == 1 and v.stride(3) == 1, "k, v: contiguous values")
        _own_elements(k)
        _own_elements(v)
        _apart(k, v, "the values")
        self._k, self._v, self._sinks, self._len = k, v, int(sinks), length
        self.slots = k.shape[1]
        item = k.element_size()
        (ka, k0, k1, k2, _, kend), (va, v0, v1, v2, _, vend) = _plain(k, item), _plain(v, item)
        self._plain = (ka, k0, k1, k2, kend, va, v0, v1, v2, vend)

    @classmethod
    def of(cls, k: torch.Tensor, v: torch.Tensor, sinks: int = 0, length: torch.Tensor | None = None) -> "TokenCache":
        """A cache over tensors that the caller holds (length: int32 [B] on the device, zeros by default)."""
        c = cls.__new__(cls)
        c._set(k, v, sinks, torch.zeros(k.shape[0], dtype=torch.int32, device=k.device) if length is None else length)
        return c

    def advance(self, n) -> "TokenCache":
        """n (an int, or int32 [B] on the device) more tokens of each stream: before they are stored.  The counts are 32 bits
        and end at 2^31 - 1: a stream that may get there (12 hours of 1600 tokens a frame, 30 frames a second) calls rebase
        now and then."""
        self._len += n
        return self

    def rebase(self, frame: int = 1) -> "TokenCache":
        """Sets counts from 2^30 on back by a whole number of rings and of ``frame`` (attend's) tokens, which changes no
        result: a ring's slots and what a query sees depend on differences of positions alone.  Others stay.  Called at
        least every 2^29 tokens (each frame is fine: it works on the device, and may be captured) a stream never ends.
        The positions of a rotation are the caller's own."""
        turn = math.lcm(self.slots - self.sinks, max(int(frame), 1))
        _need(frame >= 0 and turn <= 1 << 29 and self.slots <= 1 << 29,
              f"frame {frame}: its common multiple with the ring of {self.slots - self.sinks} slots is beyond 2^29")
        self._len -= torch.div((self._len - (1 << 30)).clamp_(min=0), turn, rounding_mode="floor") * turn
        return self


class QKNorm:
    """x / sqrt(mean(x^2) + eps) * weight for each head of the queries and keys, then ``rotary``, in one pass.

    q_weight / k_weight: [head_dim] (None: that norm is left out).  rotary: a Rotary (None: no rotation)."""

    wq, wk, rotary = _fixed("wq"), _fixed("wk"), _fixed("rotary")

    def __init__(self, head_dim: int, rotary: Rotary | None = None, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6, device=None):
        _need(1 <= head_dim <= 256, f"head_dim {head_dim}: 1 to 256")
        _need(rotary is None or rotary.dim <= head_dim, "rotary: more values than a head has")
        _need(eps >= 0, f"eps {eps}: not negative")
        for n, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            _need(w is None or w.shape == (head_dim,), f"{n}: [{head_dim}]")
        _lib.require_gpu()
        self.lib = _lib.load()
        self.device = _gpu(device)
        _need(rotary is None or rotary.device == self.device, "rotary: on another device")
        self.D, self._rotary = head_dim, rotary
        self._wq, self._wk = _floats(q_weight, self.device), _floats(k_weight, self.device)
        self.eps = float(eps)
        self._norm = (self.wq.data_ptr() if self.wq is not None else 0, self.wk.data_ptr() if self.wk is not None else 0,
                      self.eps)
        self._held = (self.wq, self.wk, *(() if rotary is None else (rotary.turns, rotary.axis)))
        self._turn = (0, 0, 0) if rotary is None else (rotary.dim, rotary.turns.data_ptr(), rotary.axis.data_ptr())
        self._rot = (0, 0) if rotary is None else (rotary.axes, LAYOUTS[rotary.layout])

    def __call__(self, q: torch.Tensor, k: torch.Tensor, pos: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None, stream=None):
        """q [B, S, Hq, D], k [B, S, Hk, D] (any strides with contiguous values, e.g. views of one product's output)
        -> (q', k').  pos: int32 [B, S, axes] ([B, S] for one axis; expanded views are fine).  q_out / k_out may be
        q / k themselves."""
        if not _here(self.device, stream):
            return _elsewhere(self.device, stream, (q, k, pos, q_out, k_out, *self._held),
                              lambda: self(q, k, pos, q_out, k_out))
        q, k, pos, turn, B, S, Hq, Hk, item = self._begin(q, k, pos)
        if q_out is None and k_out is None:
            q_out, k_out = q.new_empty(q.shape), k.new_empty(k.shape)
        else:
            q_out, k_out = (self._out(t, like, n) for t, like, n in ((q_out, q, "q_out"), (k_out, k, "k_out")))
            _apart(q_out, k, "k")
            _apart(k_out, q, "q")
            _apart(q_out, k_out, "k_out")
        if B and S:
            qa, q0, q1, q2 = q.data_ptr(), *q.stride()[:3]
            ka, k0, k1, k2 = k.data_ptr(), *k.stride()[:3]
            a = QK_PACK.pack(qa, ka, 0, q_out.data_ptr(), k_out.data_ptr(), 0, q0, q1, q2, k0, k1, k2, 0, 0, 0,
                             *q_out.stride()[:3], *k_out.stride()[:3], 0, 0, 0, *self._norm, *turn, 0, 0, B, S, Hq, Hk, self.D, 0,
                             *self._rot, 0, 0, DTYPES[q.dtype], 0)
            rc = self.lib.va_tok_qk(_raw_stream(self.device.index), a)
            if rc:
                _lib.check(rc, "va_tok_qk")
        return q_out, k_out

    def store(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor | None, cache: TokenCache,
              q_len: torch.Tensor | None = None, q_out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """The same for the last q_len[b] tokens (S at most, and by default) of cache.len[b]: -> q', with the keys and values in the
        cache.  Rows s >= q_len[b] of q_out are left as they were (zeros where the call makes it); a token whose slot a
        later one of the call takes, or whose position is negative, is not kept."""
        if not _here(self.device, stream):
            return _elsewhere(self.device, stream, (q, k, v, pos, q_len, q_out, cache.k, cache.v, cache.len, *self._held),
                              lambda: self.store(q, k, v, pos, cache, q_len, q_out))
        q, k, pos, turn, B, S, Hq, Hk, item = self._begin(q, k, pos)
        Dv = cache.v.shape[3]
        _on(v, self.device, q.dtype, "v")
        _on(cache.k, self.device, q.dtype, "the cache")
        if v.shape != (B, S, Hk, Dv):
            raise _lib.VaError(f"v {tuple(v.shape)}: {(B, S, Hk, Dv)}")
        if cache.k.shape != (B, cache.slots, Hk, self.D):
            raise _lib.VaError(f"the cache holds {tuple(cache.k.shape)}")
        if q_len is not None:
            _lens(q_len, B, self.device, "q_len")
        if q_out is None:
            q_out = (torch.empty if q_len is None else torch.zeros)(q.shape, dtype=q.dtype, device=self.device)
        else:
            q_out = self._out(q_out, q, "q_out")
        if not (B and S):
            return q_out
        va, v0, v1, v2, v3, vend = _plain(v, item)
        if v3 != 1 and Dv > 1:
            v = v.contiguous()
            va, v0, v1, v2, v3, vend = _plain(v, item)
        qa, q0, q1, q2, _, qend = _plain(q, item)
        ka, k0, k1, k2, _, kend = _plain(k, item)
        oa, o0, o1, o2, _, oend = _plain(q_out, item)
        c = cache._plain
        # (cheap first: whether two ranges of bytes meet at all)
        for n, t, at, end in (("k", k, ka, kend), ("v", v, va, vend)):
            if oa < end and at < oend:
                _apart(q_out, t, n)
        for cn, ct, cat, cend in (("the cache's keys", cache.k, c[0], c[4]), ("the cache's values", cache.v, c[5], c[9])):
            if oa < cend and cat < oend:
                _apart(q_out, ct, cn)
            for n, t, at, end in (("q", q, qa, qend), ("k", k, ka, kend), ("v", v, va, vend)):
                if at < cend and cat < end:
                    _apart(ct, t, n)
        a = QK_PACK.pack(qa, ka, va, oa, c[0], c[5], q0, q1, q2, k0, k1, k2, v0, v1, v2, o0, o1, o2, *c[1:4], *c[6:9],
                         *self._norm, *turn, 0 if q_len is None else q_len.data_ptr(), cache.len.data_ptr(), B, S, Hq, Hk, self.D, Dv,
                         *self._rot, cache.slots, cache.sinks, DTYPES[q.dtype], 0)
        rc = self.lib.va_tok_qk(_raw_stream(self.device.index), a)
        if rc:
            _lib.check(rc, "va_tok_qk")
        return q_out

    def _begin(self, q, k, pos):
        """Checks -> q, k with contiguous values, pos, (rot, turns, axis, pos, its strides), the sizes."""
        if q.dim() != 4 or k.dim() != 4:
            raise _lib.VaError(f"q {tuple(q.shape)}, k {tuple(k.shape)}: [B, S, heads, {self.D}]")
        B, S, Hq, D = q.shape
        Bk, Sk, Hk, Dk = k.shape
        if Bk != B or Sk != S or D != self.D or Dk != D:
            raise _lib.VaError(f"q {tuple(q.shape)}, k {tuple(k.shape)}: [B, S, heads, {self.D}]")
        dtype = q.dtype
        if dtype not in DTYPES:
            raise _lib.VaError(f"q is {dtype}: bfloat16 or float32")
        _on(q, self.device, dtype, "q")
        _on(k, self.device, dtype, "k")
        if B > I32_MAX or S > I32_MAX or Hq > 1 << 20 or Hk > 1 << 20:
            raise _lib.VaError("a side beyond what the kernel counts")
        if D > 1:
            q = q if q.stride(3) == 1 else q.contiguous()
            k = k if k.stride(3) == 1 else k.contiguous()
        rotary = self.rotary
        if rotary is None:
            _need(pos is None, "pos: there is no rotation")
            return q, k, None, (0, 0, 0, 0, 0, 0), B, S, Hq, Hk, q.element_size()
        if pos is None:
            raise _lib.VaError("pos: a rotation needs positions")
        _on(pos, self.device, torch.int32, "pos")
        n = rotary.axes
        pos = pos.unsqueeze(-1) if n == 1 and pos.dim() == 2 else pos
        if pos.shape != (B, S, n):
            raise _lib.VaError(f"pos {tuple(pos.shape)}: {(B, S, n)}")
        a, b, c = pos.stride()
        if n > 1 and c != 1:
            pos = pos.contiguous()
            a, b, c = pos.stride()
        return q, k, pos, (*self._turn, pos.data_ptr(), a, b), B, S, Hq, Hk, q.element_size()

    def _out(self, t, like, name):
        if t is None:
            return like.new_empty(like.shape)
        _on(t, self.device, like.dtype, name)
        if t.shape != like.shape or (t.stride(3) != 1 and self.D > 1):
            raise _lib.VaError(f"{name} {tuple(t.shape)}: {tuple(like.shape)} with contiguous values")
        _own_elements(t)
        _apart(t, like, "its input", same_ok=True)
        return t


# ------------------------------------------------------------------ attention
def _lens(t, B, dev, name):
    _on(t, dev, torch.int32, name)
    if t.dim() != 1 or t.shape[0] != B or (B > 1 and t.stride(0) != 1):
        raise _lib.VaError(f"{name} {tuple(t.shape)}: int32 [{B}]")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy of it, with contiguous values and every row 16-byte aligned."""
    a, b, c, d = t.stride()
    fine = d == 1 and not (a | b | c) % 8 and not t.data_ptr() & 15 and b < 1 << 22
    return t if fine else t.clone(memory_format=torch.contiguous_format)


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None, frame: int = 1,
           window: int = 0, sinks: int = 0, q_len: torch.Tensor | None = None, kv_len: torch.Tensor | None = None,
           out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """softmax(scale q k^T) v of q [B, S, Hq, D] over k [B, slots, Hk, D] and v [B, slots, Hk, Dv] (a TokenCache's
    tensors, or a batch of prompts), Hq a multiple of Hk: -> [B, S, Hq, Dv].

    The queries of sequence b are its last q_len[b] (S at most, and by default) of kv_len[b] (default slots) positions.  A query at
    position i sees the positions j < e = (i // frame + 1) * frame with j < sinks or j >= e - window (window 0: all of
    them): frame 1 goes token by token, frame = tokens of an image lets one image's tokens see each other, and frame 0
    (with window = sinks = 0) lets every token see every token.  With kv_len[b] > slots the tensors are rings behind
    their first ``sinks`` slots (TokenCache), and overwritten positions are not seen: for S queries over a window to see
    all of it, slots >= sinks + window + S - 1.  A query that sees nothing gets zeros; rows s >= q_len[b] of out are left
    as they were (zeros where the call makes it).  A value that is not finite makes its column of the queries that see it an
    infinity of its sign, or NaN beside NaN or the other infinity, and has no part in others.  scale: D ** -0.5 by default, positive.  D and Dv: multiples of 8 up
    to 128."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise _lib.VaError("q [B, S, Hq, D], k [B, slots, Hk, D], v [B, slots, Hk, Dv]")
    B, S, Hq, D = q.shape
    Bk, slots, Hk, Dk = k.shape
    Bv, vslots, vh, Dv = v.shape
    if Bk != B or Dk != D or (Bv, vslots, vh) != (Bk, slots, Hk):
        raise _lib.VaError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not fit")
    if Hk == 0 or Hq == 0 or Hq % Hk:
        raise _lib.VaError(f"{Hq} query heads over {Hk} key heads")
    if D % 8 or not 8 <= D <= 128 or Dv % 8 or not 8 <= Dv <= 128:
        raise _lib.VaError(f"D {D}, Dv {Dv}: multiples of 8 up to 128")
    if min(frame, window, sinks) < 0 or max(frame, window, sinks) > I32_MAX:
        raise _lib.VaError("frame, window and sinks are not negative")
    if frame == 0 and (window or sinks):
        raise _lib.VaError("frame 0 sees everything: no window, no sinks")
    if slots and sinks >= slots:
        raise _lib.VaError(f"sinks {sinks}: fewer than the {slots} slots")
    if max(B, S, slots) > I32_MAX or S * (Hq // Hk) > I32_MAX - 256:
        raise _lib.VaError("a side beyond what the kernel counts")
    scale = D ** -0.5 if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise _lib.VaError(f"scale {scale}: positive")
    dev, dtype = q.device, q.dtype
    if dtype not in DTYPES:
        raise _lib.VaError(f"q is {dtype}: bfloat16 or float32")
    _on(q, dev, dtype, "q")
    _on(k, dev, dtype, "k")
    _on(v, dev, dtype, "v")
    if q_len is not None:
        _lens(q_len, B, dev, "q_len")
    if kv_len is not None:
        _lens(kv_len, B, dev, "kv_len")
    if not _here(dev, stream):
        return _elsewhere(dev, stream, (q, k, v, q_len, kv_len, out),
                          lambda: attend(q, k, v, scale=scale, frame=frame, window=window, sinks=sinks, q_len=q_len,
                                         kv_len=kv_len, out=out))
    if out is None:
        out = (torch.empty if q_len is None else torch.zeros)((B, S, Hq, Dv), dtype=dtype, device=dev)
    else:
        _on(out, dev, dtype, "out")
        _need(out.shape == (B, S, Hq, Dv), "out: [B, S, Hq, Dv]")
        _own_elements(out)
        at = _range(out)
        for t, n in ((q, "q"), (k, "k"), (v, "v")):
            if _meet(at, _range(t)):
                _apart(out, t, n)
    if B == 0 or S == 0:
        return out
    q, k, v, o = _aligned(q), _aligned(k), _aligned(v), _aligned(out)
    lib = _lib.load()
    (q0, q1, q2, _), (k0, k1, k2, _), (v0, v1, v2, _), (o0, o1, o2, _) = q.stride(), k.stride(), v.stride(), o.stride()
    most = (q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), q0, q1, q2, k0, k1, k2, v0, v1, v2, o0, o1, o2,
            0 if q_len is None else q_len.data_ptr(), 0 if kv_len is None else kv_len.data_ptr(), scale, B, S, Hq, Hk, D, Dv,
            slots, frame, window, sinks, DTYPES[dtype])
    a = ATTN_PACK.pack(*most, 0, 0)
    n = lib.va_tok_attn_workspace_bytes(a)
    if n:
        _need(n > 0, f"va_tok_attn_workspace_bytes failed with status {n}")
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        a = ATTN_PACK.pack(*most, ws.data_ptr(), n)
    rc = lib.va_tok_attn(_raw_stream(dev.index), a)
    if rc:
        _lib.check(rc, "va_tok_attn")
    if o is not out:
        out.copy_(o)
    return out
