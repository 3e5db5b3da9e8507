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
with other ones; the cache's calls also take one Python int for all sequences.
"""

from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from .ops import _stream_ptr

_pack_write, _pack_attend, _pack_prompt = (_lib.packer(c) for c in (_lib.KvmWindowWriteArgs, _lib.KvmWindowAttendArgs, _lib.KvmWindowPromptArgs))
MAX_GROUP = 16  # query heads per kv head of the single-token calls
_BF16 = torch.bfloat16


def _rows(t: torch.Tensor, name: str, shape, dev) -> tuple:
    """[B,H,T,D] bf16 rows that are contiguous and start on 16-byte boundaries, as they lie in memory where that is so
    already: (address, strides of B, H and T, the tensor that holds them)."""
    if not isinstance(t, torch.Tensor) or t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape) if isinstance(t, torch.Tensor) else type(t)}")
    if t.dtype is not _BF16:
        raise ValueError(f"{name} must be bfloat16, got {t.dtype}")
    if t.device != dev:
        if not t.is_cuda:
            raise RuntimeError(f"{name} must live on a CUDA device (there is no CPU path)")
        raise RuntimeError(f"{name} must be on {dev}, got {t.device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("the window operators implement inference only; call them under torch.no_grad()")
    b, h, r, d = t.stride()
    p = t.data_ptr()
    if d != 1 or p & 15 or (b | h | r) & 7 or b <= 0 or h <= 0 or r <= 0:
        # a dimension of one entry is never stepped over: any stride will do there
        full = shape[3]
        b, h, r = (s if n > 1 else full for s, n in zip((b, h, r), shape))
        if (d != 1 and full > 1) or p & 15 or (b | h | r) & 7 or b <= 0 or h <= 0 or r <= 0:
            t = t.clone(memory_format=torch.contiguous_format)
            b, h, r, _ = t.stride()
            p = t.data_ptr()
    return p, b, h, r, t


def _shape4(t, name: str, want: str):
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise ValueError(f"{name} must be a {want} tensor, got {list(t.shape) if isinstance(t, torch.Tensor) else type(t)}")
    return t.shape


def _counts(x, name: str, batch: int, dev, least: int, most: int):
    """(device address or 0, number for all) of per-sequence positions or lengths."""
    if isinstance(x, torch.Tensor):
        if x.dtype is not torch.int32 or x.shape != (batch,) or not x.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 tensor of {batch} entries, got {tuple(x.shape)} {x.dtype}")
        if x.device != dev:
            raise RuntimeError(f"{name} must be on {dev}, got {x.device}")
        return x.data_ptr(), 0
    x = int(x)
    if not least <= x <= most:
        raise ValueError(f"{name} must be in [{least}, {most}], got {x}")
    return 0, x


def _int32(x, name: str) -> int:
    x = int(x)
    if not -2**31 <= x < 2**31:  # (ctypes would cut it off)
        raise ValueError(f"{name} must be a 32-bit integer, got {x}")
    return x


def _output(out, like: torch.Tensor, shape) -> torch.Tensor:
    if out is None:
        return like.new_empty(shape)
    if not isinstance(out, torch.Tensor) or (out.requires_grad and torch.is_grad_enabled()):
        raise ValueError("out must be a tensor that needs no gradient")
    if out.shape != shape or out.dtype is not _BF16 or not out.is_contiguous() or out.device != like.device or out.data_ptr() % 16:
        raise ValueError(f"out must be a contiguous, 16-byte aligned bf16 tensor {list(shape)} on {like.device}, got {list(out.shape)} {out.dtype}")
    return out


def _scale(scale, head_dim: int) -> float:
    s = 1.0 / math.sqrt(head_dim) if scale is None else float(scale)
    if not 0.0 < s < 1e38:  # (log2(e) times it is finite in fp32, too)
        raise ValueError(f"scale must be positive and below 1e38, got {s}")
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
    ``window - 1`` tokens are there.  One call takes sequences that hold equally many of them, as all do that have passed
    ``sinks + window`` tokens; others go one by one, without the zeros that ``read`` leaves behind a shorter one.)  ``window``
    None: every earlier token is visible.  ``lengths`` (int32 [B]): tokens of each sequence, S at most; what lies behind them is
    padding, is never looked at, and its output rows are zeros.
    Returns [B,T,Hq*D] (``out`` if given, which must not share memory with q, k or v)."""
    B, Hq, T, D = _shape4(q, "q", "[B,Hq,T,D]")
    _, Hkv, S, _ = _shape4(k, "k", "[B,Hkv,S,D]")
    dev = q.device
    if not q.is_cuda:
        raise RuntimeError("kvm_b200 runs on CUDA tensors only (there is no CPU path)")
    qa, ka, va = _rows(q, "q", (B, Hq, T, D), dev), _rows(k, "k", (B, Hkv, S, D), dev), _rows(v, "v", (B, Hkv, S, D), dev)
    lens = 0
    if lengths is not None:
        if not isinstance(lengths, torch.Tensor):
            raise ValueError(f"lengths must be an int32 tensor, got {type(lengths)}")
        lens, _ = _counts(lengths, "lengths", B, dev, 0, S)
    y = _output(out, q, (B, T, Hq * D))
    _call(dev, _lib.load().kvm_window_attention,
          _pack_prompt(*qa[:4], *ka[:4], *va[:4], lens, y.data_ptr(), T, S, max(S, 1) if window is None else _int32(window, "window"),
                       _int32(sinks, "sinks"), B, Hq, Hkv, D, _scale(scale, D)))
    return y


class WindowCache:
    """Keys and values of the first ``sinks`` and the last ``window`` tokens of ``batch`` sequences, in 16 bits or in 4 bits
    (4.5 with the scales; the format: include/kvm_b200.h).

    The sequences' lengths are the caller's: every call is given positions or lengths, and none of them changes any.  A token
    that is written takes the place of the one R before it for good, R being ``window`` rounded up to 16: a sequence that goes
    back by more than R - window tokens misses what they pushed out.  Calls on one cache run in the order of their streams; a
    call that writes must not overlap with another call on the same cache."""

    def __init__(self, batch: int, n_kv_heads: int, head_dim: int, *, window: int, sinks: int = 0, bits: int = 16, device="cuda"):
        self.batch, self.n_kv_heads, self.head_dim = _int32(batch, "batch"), _int32(n_kv_heads, "n_kv_heads"), _int32(head_dim, "head_dim")
        self.window, self.sinks, self.bits = _int32(window, "window"), _int32(sinks, "sinks"), _int32(bits, "bits")
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
        self._k = self._v = self._blocks = None
        if self.bits == 4:
            self._blocks = torch.zeros(n, device=dev, dtype=torch.uint8)
            c.k = self._blocks.data_ptr()
        else:  # rows in the cache's own order: sinks first, then the ring
            shape = (self.batch, self.n_kv_heads, self.rows, self.head_dim)
            self._k, self._v = (torch.zeros(shape, device=dev, dtype=_BF16) for _ in range(2))
            c.k, c.v = self._k.data_ptr(), self._v.data_ptr()
        self._addr = C.addressof(c)
        self._like = torch.empty(0, device=dev, dtype=_BF16)
        self._read_shape = (2, self.batch, self.n_kv_heads, self.sinks + self.window, self.head_dim)
        self._workspace_bytes: dict[int, int] = {}

    @property
    def k(self) -> torch.Tensor | None:
        """Keys of a 16-bit cache [B,Hkv,rows,D] in the cache's own order (include/kvm_b200.h); None for 4 bits (``read``)."""
        return self._k

    @property
    def v(self) -> torch.Tensor | None:
        """Values, as ``k``."""
        return self._v

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self._k, self._v, self._blocks) if t is not None)

    def write(self, k: torch.Tensor, v: torch.Tensor, positions, lengths=None) -> None:
        """Writes tokens ``positions[b] ...`` of every sequence: k, v [B,Hkv,T,D], of which sequence b brings the first
        ``lengths[b]`` (None: all), from memory that is not the cache's own.  A negative position leaves its sequence as it is.
        Positions stay below 2^31 - T.  Tokens that later ones of the call push out are not written."""
        T = _shape4(k, "k", "[B,Hkv,T,D]")[2]
        shape = (self.batch, self.n_kv_heads, T, self.head_dim)
        ka, va = _rows(k, "k", shape, self.device), _rows(v, "v", shape, self.device)
        p, p_all = _counts(positions, "positions", self.batch, self.device, -1, 2**31 - 1 - T)
        n, n_all = (0, T) if lengths is None else _counts(lengths, "lengths", self.batch, self.device, 0, T)
        _call(self.device, _lib.load().kvm_window_cache_write, _pack_write(self._addr, *ka[:4], *va[:4], p, n, T, p_all, n_all))

    def read(self, lengths) -> tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds of sequences of ``lengths`` tokens, in order: (k, v) [B,Hkv,sinks+window,D], the first sinks
        tokens, then the last ``window`` ones; zeros behind the last token."""
        n, n_all = _counts(lengths, "lengths", self.batch, self.device, 0, 2**31 - 1)
        k, v = self._like.new_empty(self._read_shape).unbind(0)
        _call(self.device, _lib.load().kvm_window_cache_read, self._addr, n, n_all, k.data_ptr(), v.data_ptr())
        return k, v

    def _attend(self, q, ka, va, counts, scale, out):
        Hq = _shape4(q, "q", "[B,Hq,1,D]")[1]
        qa = _rows(q, "q", (self.batch, Hq, 1, self.head_dim), self.device)
        lib = _lib.load()
        need = self._workspace_bytes.get(Hq)
        if need is None:
            if Hq <= 0 or Hq % self.n_kv_heads or Hq // self.n_kv_heads > MAX_GROUP:
                raise ValueError(f"{Hq} query heads over {self.n_kv_heads} kv heads: a multiple of them, at most {MAX_GROUP} each")
            with torch.cuda.device(self.device):
                need = self._workspace_bytes[Hq] = lib.kvm_window_attend_workspace_bytes(self._addr, Hq)
        y = _output(out, q, (self.batch, 1, Hq * self.head_dim))
        # partial results: of this call alone (calls on two streams, or in two captured graphs, do not share them)
        ws = q.new_empty(need >> 1) if need else None
        _call(self.device, lib.kvm_window_attend,
              _pack_attend(self._addr, *qa[:4], *ka, *va, counts[0], y.data_ptr(), ws.data_ptr() if need else 0, need, Hq, counts[1],
                           _scale(scale, self.head_dim)))
        return y

    def attend(self, q: torch.Tensor, lengths, *, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """One query per sequence over the cached tokens: q [B,Hq,1,D], ``lengths`` the tokens of the sequences, the query's own
        among them.  Returns [B,1,Hq*D] (``out`` if given; it may be q's own memory); a sequence of no tokens gets zeros."""
        none = (0, 0, 0, 0)
        return self._attend(q, none, none, _counts(lengths, "lengths", self.batch, self.device, 0, 2**31 - 1), scale, out)

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions, *, scale: float | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """``write`` of one token per sequence (k, v [B,Hkv,1,D]) at ``positions`` and ``attend`` of its query in one pass.  A
        sequence at position -1 is left alone and gets zeros."""
        shape = (self.batch, self.n_kv_heads, 1, self.head_dim)
        ka, va = _rows(k, "k", shape, self.device), _rows(v, "v", shape, self.device)
        return self._attend(q, ka[:4], va[:4], _counts(positions, "positions", self.batch, self.device, -1, 2**31 - 2), scale, out)


def check_status(device="cuda") -> None:
    """Synchronise and raise if a window kernel on the device, whoever called it, reported a device-side timeout since the last
    check (one word per device, cleared by the check that reports it)."""
    dev = torch.device(device)
    dev = torch.device("cuda", torch.cuda.current_device() if dev.index is None else dev.index)
    _call(dev, _lib.load().kvm_window_status)
