"""Token operators on MI355X: the layers of an attention block over the tokens of camera frames.

* ``Linear`` -- a matrix product with bias, activation and residual in its epilogue (bf16, f32 or e4m3 weights);
* ``QKNorm`` with ``Rotary`` -- the norms of queries and keys for each head and the rotation by the token's position
  on one or more axes (time, height, width) in one pass, into a ``TokenCache`` where a stream keeps one;
* ``attend`` -- attention by frames with a sliding window and first tokens that stay visible (sinks).

Each call is one launch or two of ``libva355.so`` (``va_tok_linear`` / ``va_tok_qk`` / ``va_tok_attn`` in va355.h) on
the current stream of the tensors' device, or on ``stream``; it does not synchronise, keeps nothing between calls and may
be captured into a graph.  Results are the same from call to call, bit by bit.  With ``stream``, what the call allocates
belongs to that stream, its inputs are recorded on it, and the caller orders it against the work that made them.

The operators are forward only, as every layer of this package.
"""
from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from . import _lib
from .seg import VA_DTYPE_BF16, VA_DTYPE_F32, split3_bf16, w8_order

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


# ------------------------------------------------------------------ what every call checks
def _need(ok: bool, what: str) -> None:
    if not ok:
        raise _lib.VaError(what)


def _on(t: torch.Tensor, dev: torch.device, dtype, name: str) -> None:
    if t.device != dev:
        raise _lib.VaError(f"{name} is on {t.device}, not on {dev}")
    if t.dtype != dtype:
        raise _lib.VaError(f"{name} is {t.dtype}, not {dtype}")


def _range(t: torch.Tensor) -> tuple[int, int]:
    """The bytes between a tensor's first and last element (0, 0: it has none)."""
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


def _apart(out: torch.Tensor, t: torch.Tensor | None, name: str, same_ok: bool = False) -> None:
    """Refuses an output that overlaps an input (same_ok: unless it is that very tensor)."""
    if t is None:
        return
    (a, b), (c, d) = _range(out), _range(t)
    if a < d and c < b and not (same_ok and out.data_ptr() == t.data_ptr() and out.shape == t.shape and
                                out.stride() == t.stride() and out.dtype == t.dtype) \
            and not _interleaved(out, t):
        raise _lib.VaError(f"the output overlaps {name}")


def _own_elements(out: torch.Tensor) -> None:
    """Refuses an output whose elements share memory (an expanded tensor)."""
    at = 1
    for s, n in sorted((s, n) for n, s in zip(out.shape, out.stride()) if n > 1):
        _need(s >= at, "the output's elements overlap")
        at = s * n


class _Launch:
    """The device and stream of one call; what it allocates inside belongs to that stream."""

    def __init__(self, dev: torch.device, stream, inputs):
        self.scope = None
        if dev.type != "cuda":
            raise _lib.VaError(f"the token operators need tensors on the GPU, not on {dev}")
        if stream is None:
            if dev.index != torch.cuda.current_device():
                self.scope = torch.cuda.device(dev)
                self.scope.__enter__()
            self.ptr = torch.cuda.current_stream(dev).cuda_stream
            return
        self.ptr = _lib.stream_ptr(stream, dev)
        self.scope = contextlib.ExitStack()
        self.scope.enter_context(torch.cuda.device(dev))
        self.scope.enter_context(torch.cuda.stream(stream))
        for t in inputs:
            if t is not None:
                t.record_stream(stream)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        if self.scope is not None:
            self.scope.__exit__(*exc)
        return False


# ------------------------------------------------------------------ matrix product
class Linear:
    """y = act(x w^T + bias) + residual, the weights packed once.

    weight: [N, K].  dtype "bf16" (bf16 tensors), "f32" (float tensors; every product as six exact bf16 term products,
    float sums) or "w8a16" (bf16 tensors, e4m3 weight bytes with one float scale per row: quantised here as the
    convolutions' are, or given as float8_e4m3fn values with ``scale`` [N]).  bias: [N].  act: None, "silu", "gelu",
    "gelu_tanh" or "relu"."""

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
        if device is None:
            device = weight.device if weight.device.type == "cuda" else torch.device("cuda", torch.cuda.current_device())
        self.device = torch.device(device)
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.lib = _lib.load()
        self.N, self.K, self.dtype = N, K, dtype
        self.tdtype = torch.float32 if dtype == "f32" else torch.bfloat16
        Np, Kp = -(-N // 64) * 64, -(-K // 64) * 64

        def padded(t):
            p = torch.zeros(Np, Kp, dtype=t.dtype, device=self.device)
            p[:N, :K] = t
            return p

        w, self.wscale = weight.detach().to(self.device), None
        if dtype == "w8a16":
            if scale is None:
                from .seg import F8_MAX
                w = w.float()
                amax = w.abs().amax(1)
                scale = torch.where(amax > 0, amax / F8_MAX, torch.ones_like(amax))
                w = (w / scale[:, None]).clamp(-F8_MAX, F8_MAX).to(torch.float8_e4m3fn)
            self.wscale = torch.ones(Np, dtype=torch.float32, device=self.device)
            self.wscale[:N] = scale.detach().to(self.device, torch.float32)
            self.w = w8_order(padded(w.view(torch.uint8)))
        elif dtype == "f32":
            self.w = split3_bf16(padded(w.float()))
        else:
            self.w = padded(w.to(torch.bfloat16))
        self.bias = None if bias is None else bias.detach().to(self.device, torch.float32).contiguous()
        self._args = LinearArgs(w=self.w.data_ptr(), wscale=self.wscale.data_ptr() if self.wscale is not None else None,
                                bias=self.bias.data_ptr() if bias is not None else None, N=N, K=K, Npad=Np, Kpad=Kp,
                                dtype=VA_DTYPE_F32 if dtype == "f32" else VA_DTYPE_BF16, w8=int(dtype == "w8a16"),
                                act=ACTS[act])

    def args(self, x: torch.Tensor, out: torch.Tensor, residual: torch.Tensor | None = None) -> LinearArgs:
        """The va_tok_linear_args of a call on [M, K] rows (for an op list: VA_OP_TOK_LINEAR); they point into these
        tensors, which the caller keeps."""
        a = LinearArgs.from_buffer_copy(self._args)
        a.x, a.y, a.M = x.data_ptr(), out.data_ptr(), x.shape[0]
        one = a.M <= 1  # a single row's stride says nothing
        a.ldx, a.ldy = self.K if one else x.stride(0), self.N if one else out.stride(0)
        if residual is not None:
            a.res, a.ldr = residual.data_ptr(), self.N if one else residual.stride(0)
        a.out_f32 = int(out.dtype == torch.float32 and self.tdtype != torch.float32)
        return a

    def __call__(self, x: torch.Tensor, residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 stream=None) -> torch.Tensor:
        """x [..., K] -> [..., N].  residual [..., N] is added after the activation.  out: bf16 or (for the bf16 forms)
        float; it may be the residual itself, and must not overlap x."""
        _on(x, self.device, self.tdtype, "x")
        lead = x.shape[:-1]
        _need(x.dim() >= 1 and x.shape[-1] == self.K, f"x {tuple(x.shape)}: [..., {self.K}]")
        with _Launch(self.device, stream, (x, residual, out, self.w)) as at:
            x2 = self._rows(x, self.K)
            _need(x2.shape[0] <= I32_MAX, "more rows than 32 bits count")
            r2 = None
            if residual is not None:
                _on(residual, self.device, self.tdtype, "residual")
                _need(residual.shape == (*lead, self.N), f"residual {tuple(residual.shape)}: {(*lead, self.N)}")
                r2 = self._rows(residual, self.N)
            if out is None:
                out = torch.empty((*lead, self.N), dtype=self.tdtype, device=self.device)
                o2 = out.view(-1, self.N)
            else:
                _need(out.dtype in (self.tdtype, torch.float32), f"out is {out.dtype}")
                _on(out, self.device, out.dtype, "out")
                _need(out.shape == (*lead, self.N), f"out {tuple(out.shape)}: {(*lead, self.N)}")
                _own_elements(out)
                try:
                    o2 = out.view(-1, self.N) if out.numel() else out.reshape(-1, self.N)
                except RuntimeError:
                    o2 = None
                _need(o2 is not None and (self.N == 1 or o2.numel() == 0 or o2.stride(1) == 1),
                      "out: rows of a common stride with contiguous values")
                _apart(o2, x, "x")
                _apart(o2, r2, "the residual", same_ok=True)
            if x2.shape[0]:
                _lib.check(self.lib.va_tok_linear(at.ptr, ctypes.byref(self.args(x2, o2, r2))), "va_tok_linear")
        return out

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
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.turns = torch.tensor([base ** -v / (2 * math.pi) for v in e], dtype=torch.float64, device=self.device)
        self.axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], dtype=torch.int32,
                                 device=self.device)


class TokenCache:
    """Keys and values of the last tokens of B streams, and of their first ``sinks`` tokens.

    k [B, slots, heads, D], v [B, slots, heads, Dv], len [B] (int32, on the device): tokens seen so far.  Position p is
    kept in slot p while p < slots; later ones take the slots behind the sinks in turn."""

    def __init__(self, B: int, slots: int, heads: int, head_dim: int, v_dim: int | None = None, sinks: int = 0,
                 dtype: str = "bf16", device=None):
        _need(dtype in ("bf16", "f32"), f"dtype {dtype!r}: bf16 or f32")
        _need(min(B, slots, heads, head_dim) > 0, "B, slots, heads and head_dim are positive")
        _lib.require_gpu()
        t, dev = torch.float32 if dtype == "f32" else torch.bfloat16, device if device is not None else "cuda"
        self._set(torch.zeros(B, slots, heads, head_dim, dtype=t, device=dev),
                  torch.zeros(B, slots, heads, v_dim or head_dim, dtype=t, device=dev), sinks,
                  torch.zeros(B, dtype=torch.int32, device=dev))

    def _set(self, k, v, sinks, length):
        _need(k.dim() == 4 and v.dim() == 4 and k.shape[:3] == v.shape[:3] and k.dtype == v.dtype and k.device == v.device,
              "k [B, slots, heads, D] and v [B, slots, heads, Dv] of one type")
        _need(0 <= sinks < k.shape[1], f"sinks {sinks}: fewer than the {k.shape[1]} slots")
        _on(length, k.device, torch.int32, "length")
        _need(length.shape == (k.shape[0],) and length.is_contiguous(), "length: [B]")
        self.k, self.v, self.sinks, self.len = k, v, int(sinks), length
        self.slots = k.shape[1]

    @classmethod
    def of(cls, k: torch.Tensor, v: torch.Tensor, sinks: int = 0, length: torch.Tensor | None = None) -> "TokenCache":
        """A cache over tensors that the caller holds (length: int32 [B] on the device, zeros by default)."""
        c = cls.__new__(cls)
        c._set(k, v, sinks, torch.zeros(k.shape[0], dtype=torch.int32, device=k.device) if length is None else length)
        return c

    def advance(self, n) -> "TokenCache":
        """n (an int, or int32 [B] on the device) more tokens of each stream: before they are stored."""
        self.len += n
        return self


class QKNorm:
    """x / sqrt(mean(x^2) + eps) * weight for each head of the queries and keys, then ``rotary``, in one pass.

    q_weight / k_weight: [head_dim] (None: that norm is left out).  rotary: a Rotary (None: no rotation)."""

    def __init__(self, head_dim: int, rotary: Rotary | None = None, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6, device=None):
        _need(1 <= head_dim <= 256, f"head_dim {head_dim}: 1 to 256")
        _need(rotary is None or rotary.dim <= head_dim, "rotary: more values than a head has")
        _need(eps >= 0, f"eps {eps}: not negative")
        for n, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            _need(w is None or w.shape == (head_dim,), f"{n}: [{head_dim}]")
        _lib.require_gpu()
        self.lib = _lib.load()
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        _need(rotary is None or rotary.device == self.device, "rotary: on another device")
        self.D, self.rotary = head_dim, rotary
        self.wq, self.wk = (None if w is None else w.detach().to(self.device, torch.float32).contiguous()
                            for w in (q_weight, k_weight))
        a = self._args = QKArgs(D=head_dim, eps=eps)
        if self.wq is not None:
            a.q_weight = self.wq.data_ptr()
        if self.wk is not None:
            a.k_weight = self.wk.data_ptr()
        if rotary is not None:
            a.rot, a.layout, a.turns, a.axis = rotary.dim, LAYOUTS[rotary.layout], rotary.turns.data_ptr(), rotary.axis.data_ptr()

    def __call__(self, q: torch.Tensor, k: torch.Tensor, pos: torch.Tensor | None = None,
                 q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None, stream=None):
        """q [B, S, Hq, D], k [B, S, Hk, D] (any strides with contiguous values, e.g. views of one product's output)
        -> (q', k').  pos: int32 [B, S, axes] ([B, S] for one axis; expanded views are fine).  q_out / k_out may be
        q / k themselves."""
        with _Launch(self.device, stream, (q, k, pos, q_out, k_out)) as at:
            a, q, k = self._begin(q, k, pos)
            q_out, k_out = (self._out(t, like, n) for t, like, n in ((q_out, q, "q_out"), (k_out, k, "k_out")))
            self._tell(a, q, k, None, q_out, k_out, None)
            _apart(q_out, k, "k")
            _apart(k_out, q, "q")
            _apart(q_out, k_out, "k_out")
            if q.shape[0] * q.shape[1]:
                _lib.check(self.lib.va_tok_qk(at.ptr, ctypes.byref(a)), "va_tok_qk")
        return q_out, k_out

    def store(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor | None, cache: TokenCache,
              q_len: torch.Tensor | None = None, q_out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
        """The same for the last q_len[b] tokens (default S) of cache.len[b]: -> q', with the keys and values in the
        cache.  Rows s >= q_len[b] of q_out are left as they were; a token whose slot a later one of the call takes,
        or whose position is negative, is not kept."""
        with _Launch(self.device, stream, (q, k, v, pos, q_len, q_out, cache.k, cache.v, cache.len)) as at:
            a, q, k = self._begin(q, k, pos)
            B, S, Hk = k.shape[:3]
            _on(v, self.device, q.dtype, "v")
            Dv = cache.v.shape[3]
            _need(v.shape == (B, S, Hk, Dv), f"v {tuple(v.shape)}: {(B, S, Hk, Dv)}")
            v = v if v.stride(3) == 1 or Dv == 1 else v.contiguous()
            _on(cache.k, self.device, q.dtype, "the cache")
            _need(cache.k.shape[0] == B and cache.k.shape[2:] == (Hk, self.D), f"the cache holds {tuple(cache.k.shape)}")
            _need(cache.k.stride(3) == 1 and cache.v.stride(3) == 1, "the cache's values are not contiguous")
            _own_elements(cache.k)
            _own_elements(cache.v)
            q_out = self._out(q_out, q, "q_out", torch.zeros if q_len is not None else torch.empty)
            if q_len is not None:
                _lens(q_len, B, self.device, "q_len")
                a.q_len = q_len.data_ptr()
            a.kv_len, a.slots, a.sinks = cache.len.data_ptr(), cache.slots, cache.sinks
            self._tell(a, q, k, v, q_out, cache.k, cache.v)
            for t, n in ((cache.k, "the cache's keys"), (cache.v, "the cache's values")):
                _apart(q_out, t, n)
                for u, m in ((q, "q"), (k, "k"), (v, "v")):
                    _apart(t, u, m)
            _apart(q_out, k, "k")
            _apart(q_out, v, "v")
            _apart(cache.k, cache.v, "the cache's values")
            if B * S:
                _lib.check(self.lib.va_tok_qk(at.ptr, ctypes.byref(a)), "va_tok_qk")
        return q_out

    def _begin(self, q, k, pos):
        a = QKArgs.from_buffer_copy(self._args)
        _need(q.dim() == 4 and k.dim() == 4 and q.shape[:2] == k.shape[:2] and q.shape[3] == k.shape[3] == self.D,
              f"q {tuple(q.shape)}, k {tuple(k.shape)}: [B, S, heads, {self.D}]")
        _need(q.dtype in DTYPES, f"q is {q.dtype}: bfloat16 or float32")
        _on(q, self.device, q.dtype, "q")
        _on(k, self.device, q.dtype, "k")
        B, S = q.shape[:2]
        _need(max(B, S) <= I32_MAX and max(q.shape[2], k.shape[2]) <= 1 << 20, "a side beyond what the kernel counts")
        q, k = (t if t.stride(3) == 1 or self.D == 1 else t.contiguous() for t in (q, k))
        a.B, a.S, a.Hq, a.Hk, a.dtype = B, S, q.shape[2], k.shape[2], DTYPES[q.dtype]
        if self.rotary is not None:
            n = self.rotary.axes
            _need(pos is not None, "pos: a rotation needs positions")
            _on(pos, self.device, torch.int32, "pos")
            pos = pos.unsqueeze(-1) if pos.dim() == 2 and n == 1 else pos
            _need(pos.shape == (B, S, n), f"pos {tuple(pos.shape)}: {(B, S, n)}")
            if n > 1 and pos.stride(2) != 1:
                pos = pos.contiguous()
            a.pos, a.pos_sb, a.pos_ss, a.axes = pos.data_ptr(), pos.stride(0), pos.stride(1), n
            self._hold = None
        else:
            _need(pos is None, "pos: there is no rotation")
        a._keep = (q, k, pos)  # copies live as long as the arguments
        return a, q, k

    def _out(self, t, like, name, new=torch.empty):
        if t is None:
            return new(like.shape, dtype=like.dtype, device=like.device)
        _on(t, self.device, like.dtype, name)
        _need(t.shape == like.shape and (t.stride(3) == 1 or self.D == 1),
              f"{name} {tuple(t.shape)}: {tuple(like.shape)} with contiguous values")
        _own_elements(t)
        _apart(t, like, "its input", same_ok=True)
        return t

    def _tell(self, a, q, k, v, q_out, k_out, v_out):
        for n, t in (("q", q), ("k", k), ("v", v)):
            if t is not None:
                setattr(a, n, t.data_ptr())
                for i, d in enumerate(("sb", "ss", "sh")):
                    setattr(a, f"{n}_{d}", t.stride(i))
        for n, t in (("q", q_out), ("k", k_out), ("v", v_out)):
            if t is not None:
                setattr(a, n + "_out", t.data_ptr())
                for i, d in enumerate(("sb", "ss", "sh")):
                    setattr(a, f"{n}o_{d}", t.stride(i))
        if v is not None:
            a.Dv = v.shape[3]


# ------------------------------------------------------------------ attention
def _lens(t, B, dev, name):
    _on(t, dev, torch.int32, name)
    _need(t.shape == (B,) and (B <= 1 or t.stride(0) == 1), f"{name} {tuple(t.shape)}: int32 [{B}]")


def _aligned(t: torch.Tensor) -> bool:
    """Contiguous values, every row 16-byte aligned."""
    return t.stride(3) == 1 and not (t.stride(0) | t.stride(1) | t.stride(2)) % 8 and not t.data_ptr() & 15


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: float | None = None, frame: int = 1,
           window: int = 0, sinks: int = 0, q_len: torch.Tensor | None = None, kv_len: torch.Tensor | None = None,
           out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """softmax(scale q k^T) v of q [B, S, Hq, D] over k [B, slots, Hk, D] and v [B, slots, Hk, Dv] (a TokenCache's
    tensors, or a batch of prompts), Hq a multiple of Hk: -> [B, S, Hq, Dv].

    The queries of sequence b are its last q_len[b] (default S) of kv_len[b] (default slots) positions.  A query at
    position i sees the positions j < e = (i // frame + 1) * frame with j < sinks or j >= e - window (window 0: all of
    them): frame 1 goes token by token, frame = tokens of an image lets one image's tokens see each other, and frame 0
    (with window = sinks = 0) lets every token see every token.  With kv_len[b] > slots the tensors are rings behind
    their first ``sinks`` slots (TokenCache), and overwritten positions are not seen: for S queries over a window to see
    all of it, slots >= sinks + window + S - 1.  A query that sees nothing gets zeros; rows s >= q_len[b] of out are left
    as they were (zeros where the call makes it).  scale: D ** -0.5 by default, positive.  D and Dv: multiples of 8 up
    to 128."""
    _need(q.dim() == 4 and k.dim() == 4 and v.dim() == 4, "q [B, S, Hq, D], k [B, slots, Hk, D], v [B, slots, Hk, Dv]")
    B, S, Hq, D = q.shape
    slots, Hk, Dv = k.shape[1], k.shape[2], v.shape[3]
    _need(k.shape == (B, slots, Hk, D) and v.shape == (B, slots, Hk, Dv),
          f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not fit")
    _need(Hk > 0 and Hq > 0 and Hq % Hk == 0, f"{Hq} query heads over {Hk} key heads")
    _need(D % 8 == 0 and 8 <= D <= 128 and Dv % 8 == 0 and 8 <= Dv <= 128, f"D {D}, Dv {Dv}: multiples of 8 up to 128")
    _need(frame >= 0 and window >= 0 and sinks >= 0 and max(frame, window, sinks) <= I32_MAX,
          "frame, window and sinks are not negative")
    _need(frame > 0 or window == sinks == 0, "frame 0 sees everything: no window, no sinks")
    _need(slots == 0 or sinks < slots, f"sinks {sinks}: fewer than the {slots} slots")
    _need(max(B, S, slots) <= I32_MAX and S * (Hq // Hk) <= I32_MAX - 256, "a side beyond what the kernel counts")
    scale = D ** -0.5 if scale is None else float(scale)
    _need(0 < scale < math.inf, f"scale {scale}: positive")
    _need(q.dtype in DTYPES, f"q is {q.dtype}: bfloat16 or float32")
    dev = q.device
    _on(k, dev, q.dtype, "k")
    _on(v, dev, q.dtype, "v")
    if q_len is not None:
        _lens(q_len, B, dev, "q_len")
    if kv_len is not None:
        _lens(kv_len, B, dev, "kv_len")
    lib = _lib.load()
    with _Launch(dev, stream, (q, k, v, q_len, kv_len, out)) as at:
        if out is None:
            out = (torch.empty if q_len is None else torch.zeros)((B, S, Hq, Dv), dtype=q.dtype, device=dev)
        else:
            _on(out, dev, q.dtype, "out")
            _need(out.shape == (B, S, Hq, Dv), f"out {tuple(out.shape)}: {(B, S, Hq, Dv)}")
            _own_elements(out)
            for t, n in ((q, "q"), (k, "k"), (v, "v")):
                _apart(out, t, n)
        if out.numel() == 0:
            return out
        q, k, v = (t if _aligned(t) else t.contiguous() for t in (q, k, v))
        q, k, v = (t if _aligned(t) else t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
        o = out if _aligned(out) else out.clone(memory_format=torch.contiguous_format)
        a = AttnArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), *q.stride()[:3], *k.stride()[:3],
                     *v.stride()[:3], *o.stride()[:3], None if q_len is None else q_len.data_ptr(),
                     None if kv_len is None else kv_len.data_ptr(), scale, B, S, Hq, Hk, D, Dv, slots, frame, window, sinks,
                     DTYPES[q.dtype], None, 0)
        n = lib.va_tok_attn_workspace_bytes(ctypes.byref(a))
        if n:
            _need(n > 0, f"va_tok_attn_workspace_bytes failed with status {n}")
            ws = torch.empty(n, dtype=torch.uint8, device=dev)
            a.ws, a.ws_bytes = ws.data_ptr(), n
        _lib.check(lib.va_tok_attn(at.ptr, ctypes.byref(a)), "va_tok_attn")
        if o is not out:
            out.copy_(o)
    return out
