"""Sliding-window attention with sinks: prompts, and single tokens over a cache in 16 or 4 bits.

A token at position p sees position j if ``j <= p and (j > p - window or j < sinks)``: the last ``window`` tokens, itself among
them, and the first ``sinks`` tokens of its sequence.  These are the operators of the sliding-window layers that models put
between their KVM layers (the reference's own such mixers, model/swa_mixer.py, call library attention):

    y = window_attention(q, k, v, window=4096, sinks=4)                      # a prompt
    cache = WindowCache(batch, n_kv_heads, head_dim, window=4096, sinks=4, bits=4)
    cache.write(k, v, 0)                                                     # quantised as it is written
    y = cache.step(q1, k1, v1, positions)                                    # one token per sequence, written on the way
    k, v = cache.read(lengths)                                               # in order, for the next chunk of a prompt

All of it is bf16, on CUDA devices, inference only.  Calls only enqueue kernels on the current stream of the tensors' device;
nothing is read back.  Positions and lengths are device tensors (int32, [batch]), so that a captured graph can be replayed
with other ones, or one Python int for all sequences.
"""

from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from ._lib import KvmTensor4
from .ops import _stream_ptr

MAX_GROUP = 16  # query heads per kv head of the single-token calls


def _rows(t: torch.Tensor, name: str, shape, dev) -> torch.Tensor:
    """[B,H,T,D] bf16 rows that are contiguous and start on 16-byte boundaries: a view where that is so already."""
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape) if isinstance(t, torch.Tensor) else type(t)}")
    if t.dtype is not torch.bfloat16:
        raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on a CUDA device (there is no CPU path)")
    if t.device != dev:
        raise RuntimeError(f"{name} must be on {dev}, got {t.device}")
    if torch.is_grad_enabled() and t.requires_grad:
        raise ValueError("the window operators implement inference only; call them under torch.no_grad()")
    st = t.stride()
    # (a dimension of one entry is never stepped over)
    if st[3] != 1 or t.data_ptr() % 16 or any(s % 8 or s <= 0 for s, n in zip(st[:3], t.shape) if n > 1):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _arg(t: torch.Tensor) -> KvmTensor4:
    st = t.stride()
    return KvmTensor4(t.data_ptr(), *(s if n > 1 else 0 for s, n in zip(st[:3], t.shape)))


def _counts(x, name: str, batch: int, dev, least: int, most: int):
    """(device address or None, number for all) of per-sequence positions or lengths."""
    if isinstance(x, torch.Tensor):
        if x.dtype is not torch.int32 or tuple(x.shape) != (batch,) or not x.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor of {batch} entries, got {tuple(x.shape)} {x.dtype}")
        if x.device != dev:
            raise RuntimeError(f"{name} must be on {dev}, got {x.device}")
        return x.data_ptr(), 0
    x = int(x)
    if not least <= x <= most:
        raise ValueError(f"{name} must be in [{least}, {most}], got {x}")
    return None, x


def _output(out, shape, dev) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, device=dev, dtype=torch.bfloat16)
    if tuple(out.shape) != tuple(shape) or out.dtype is not torch.bfloat16 or not out.is_contiguous() or out.device != dev or out.data_ptr() % 16:
        raise ValueError(f"out must be a contiguous, 16-byte aligned bf16 tensor {list(shape)} on {dev}, got {list(out.shape)} {out.dtype}")
    return out


def _scale(scale, head_dim: int) -> float:
    s = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    if not 0.0 < s < math.inf:
        raise ValueError(f"scale must be positive and finite, got {s}")
    return s


def _call(dev, fn, *args):
    """``fn(*args, stream)`` with the tensors' device as the current one."""
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream_ptr(dev))
    else:
        rc = fn(*args, _stream_ptr(dev))
    if rc:
        _lib.check(rc)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int | None, sinks: int = 0,
                     scale: float | None = None, lengths: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a prompt, or of a chunk of one behind earlier tokens.

    q [B,Hq,T,D], k, v [B,Hkv,S,D] with S >= T; query t stands at position S - T + t.  (The earlier tokens of a chunk may be
    what ``WindowCache.read`` returns: positions only count relative to each other, as long as the sinks and the last
    ``window - 1`` tokens are there.)  ``window`` None: every earlier token is visible.  ``lengths`` (int32 [B]): tokens of each
    sequence, S at most; what lies behind them is padding, is never looked at, and its output rows are zeros.
    Returns [B,T,Hq*D] (``out`` if given)."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise ValueError(f"{name} must be a [B,H,T,D] tensor, got {list(t.shape) if isinstance(t, torch.Tensor) else type(t)}")
    B, Hq, T, D = q.shape
    Hkv, S = k.size(1), k.size(2)
    dev = q.device
    window = max(S, 1) if window is None else int(window)
    q, k, v = _rows(q, "q", (B, Hq, T, D), dev), _rows(k, "k", (B, Hkv, S, D), dev), _rows(v, "v", (B, Hkv, S, D), dev)
    sc = _scale(scale, D)
    lens = None
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor):
            raise ValueError(f"lengths must be an int32 tensor, got {type(lengths)}")
        lens, _ = _counts(lengths, "lengths", B, dev, 0, S)
    y = _output(out, (B, T, Hq * D), dev)
    _call(dev, _lib.load().kvm_window_attention, B, Hq, Hkv, D, T, S, _arg(q), _arg(k), _arg(v), window, int(sinks), sc, lens, y.data_ptr())
    return y


class WindowCache:
    """Keys and values of the first ``sinks`` and the last ``window`` tokens of ``batch`` sequences, in 16 bits or in 4 bits
    (4.5 with the scales; the format: include/kvm_b200.h).

    The sequences' lengths are the caller's: every call is given positions or lengths, and none of them changes any.  Calls on
    one cache run in the order of their streams; a call that writes must not overlap with another call on the same cache."""

    def __init__(self, batch: int, n_kv_heads: int, head_dim: int, *, window: int, sinks: int = 0, bits: int = 16, device="cuda"):
        self.batch, self.n_kv_heads, self.head_dim = int(batch), int(n_kv_heads), int(head_dim)
        self.window, self.sinks, self.bits = int(window), int(sinks), int(bits)
        dev = torch.device(device)
        if dev.type != "cuda":
            raise RuntimeError("kvm_b200 runs on CUDA devices only (there is no CPU path)")
        lib = _lib.load()
        c = self._c = _lib.KvmWindowCache(self.batch, self.n_kv_heads, self.head_dim, self.window, self.sinks, self.bits, None, None)
        n = lib.kvm_window_cache_bytes(C.byref(c))
        if not n:
            raise ValueError(lib.kvm_last_error_string().decode())
        self.device = dev = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
        self.rows = -(-self.sinks // 16) * 16 + -(-self.window // 16) * 16
        self.k = self.v = self._blocks = None
        if self.bits == 4:
            self._blocks = torch.zeros(n, device=dev, dtype=torch.uint8)
            c.k = self._blocks.data_ptr()
        else:  # rows in the cache's own order: sinks first, then the ring
            shape = (self.batch, self.n_kv_heads, self.rows, self.head_dim)
            self.k, self.v = (torch.zeros(shape, device=dev, dtype=torch.bfloat16) for _ in range(2))
            c.k, c.v = self.k.data_ptr(), self.v.data_ptr()
        self._arg = C.byref(c)
        self._workspace_bytes: dict[int, int] = {}

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self._blocks) if t is not None)

    def write(self, k: torch.Tensor, v: torch.Tensor, positions, lengths=None) -> None:
        """Writes tokens ``positions[b] ...`` of every sequence: k, v [B,Hkv,T,D], of which sequence b brings the first
        ``lengths[b]`` (None: all).  A negative position leaves its sequence as it is.  Positions stay below 2^31 - T.  Tokens that
        later ones of the call push out are not written."""
        if not isinstance(k, torch.Tensor) or k.dim() != 4:
            raise ValueError(f"k must be a [B,Hkv,T,D] tensor, got {list(k.shape) if isinstance(k, torch.Tensor) else type(k)}")
        shape = (self.batch, self.n_kv_heads, k.size(2), self.head_dim)
        k, v = _rows(k, "k", shape, self.device), _rows(v, "v", shape, self.device)
        T = shape[2]
        p = _counts(positions, "positions", self.batch, self.device, -1, 2**31 - 1 - T)
        n = _counts(T if lengths is None else lengths, "lengths", self.batch, self.device, 0, T)
        _call(self.device, _lib.load().kvm_window_cache_write, self._arg, _arg(k), _arg(v), T, *p, *n)

    def read(self, lengths) -> tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds of sequences of ``lengths`` tokens, in order: (k, v) [B,Hkv,sinks+window,D], the first sinks
        tokens, then the last ``window`` ones; zeros behind the last token."""
        n = _counts(lengths, "lengths", self.batch, self.device, 0, 2**31 - 1)
        shape = (self.batch, self.n_kv_heads, self.sinks + self.window, self.head_dim)
        k, v = (torch.empty(shape, device=self.device, dtype=torch.bfloat16) for _ in range(2))
        _call(self.device, _lib.load().kvm_window_cache_read, self._arg, *n, k.data_ptr(), v.data_ptr())
        return k, v

    def _attend(self, q, new, counts, scale, out):
        if not isinstance(q, torch.Tensor) or q.dim() != 4:
            raise ValueError(f"q must be a [B,Hq,1,D] tensor, got {list(q.shape) if isinstance(q, torch.Tensor) else type(q)}")
        dev, Hq = self.device, q.size(1)
        q = _rows(q, "q", (self.batch, Hq, 1, self.head_dim), dev)
        lib = _lib.load()
        need = self._workspace_bytes.get(Hq)
        if need is None:
            if Hq <= 0 or Hq % self.n_kv_heads or Hq // self.n_kv_heads > MAX_GROUP:
                raise ValueError(f"{Hq} query heads over {self.n_kv_heads} kv heads: a multiple of them, at most {MAX_GROUP} each")
            need = self._workspace_bytes[Hq] = lib.kvm_window_attend_workspace_bytes(self._arg, Hq)
        y = _output(out, (self.batch, 1, Hq * self.head_dim), dev)
        # partial results: of this call alone (calls on two streams, or in two captured graphs, do not share them)
        ws = torch.empty(need, device=dev, dtype=torch.uint8)
        none = KvmTensor4(None, 0, 0, 0)
        kn, vn = (_arg(t) for t in new) if new else (none, none)
        _call(dev, lib.kvm_window_attend, self._arg, Hq, _arg(q), kn, vn, *counts, _scale(scale, self.head_dim), y.data_ptr(), ws.data_ptr(), need)
        return y

    def attend(self, q: torch.Tensor, lengths, *, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """One query per sequence over the cached tokens: q [B,Hq,1,D], ``lengths`` the tokens of the sequences, the query's own
        among them.  Returns [B,1,Hq*D]; a sequence of no tokens gets zeros."""
        return self._attend(q, None, _counts(lengths, "lengths", self.batch, self.device, 0, 2**31 - 1), scale, out)

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions, *, scale: float | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """``write`` of one token per sequence (k, v [B,Hkv,1,D]) at ``positions`` and ``attend`` of its query in one pass.  A
        sequence at position -1 is left alone and gets zeros."""
        shape = (self.batch, self.n_kv_heads, 1, self.head_dim)
        new = _rows(k, "k", shape, self.device), _rows(v, "v", shape, self.device)
        return self._attend(q, new, _counts(positions, "positions", self.batch, self.device, -1, 2**31 - 2), scale, out)


def check_status(device="cuda") -> None:
    """Synchronise and raise if a window kernel on the device reported a device-side timeout since the last check."""
    dev = torch.device(device)
    dev = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
    _call(dev, _lib.load().kvm_window_status)
