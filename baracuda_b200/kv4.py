"""Plans of the attention step over a paged 4-bit cache: norms and rotation of queries and keys, append, read, attention.

They stand between the quantized linear plans of a decoder layer: the qkv projection (`QuantizedLinearPlan`) leaves bf16
queries, keys and values in one matrix, `QkNormRopePlan` turns them and fills the cache, `Kv4AttentionPlan` reads it, and its
output feeds the output projection.  Storage, formulas and statuses are in include/baracuda_kernels_q.h.

Matrices are 2-D torch CUDA tensors with unit column stride, `[tokens, heads * head_dim]`; the row pitch is the tensor's own, so
columns of a wider matrix are passed as slices.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import _lib
from .plans import _check_backend
from .vocab import (
    BufferTooSmall,
    InvalidProblem,
    PlanPreference,
    Unsupported,
    WorkspaceTooSmall,
    status_to_result,
)

_BF16 = torch.bfloat16


# A decode step is a few microseconds on the GPU, so a call costs the host little: every tensor is asked once for each property.
def _device_of(t: Optional[torch.Tensor], name: str) -> int:
    device = -1 if t is None else t.get_device()
    if device < 0:
        raise InvalidProblem(f"{name}: expected a device buffer")
    return device


def _matrix(t: Optional[torch.Tensor], rows: int, cols: int, name: str, device: int) -> tuple:
    """(pointer, row pitch) of a bf16 matrix of at least `rows` rows and exactly `cols` columns on `device`."""
    if t is None:
        raise InvalidProblem(f"{name} is required")
    if t.dtype is not _BF16 or t.get_device() != device:
        raise InvalidProblem(f"{name}: expected a bfloat16 device matrix, on the device of the others")
    shape = t.shape
    if len(shape) != 2 or shape[1] != cols:
        raise InvalidProblem(f"{name}: expected [{rows}, {cols}], got {list(shape)}")
    ld, unit = t.stride()
    if shape[0] < rows:
        raise BufferTooSmall(f"{name}: need {rows} rows, got {shape[0]}")
    if unit != 1 and cols > 1:
        raise InvalidProblem(f"{name}: expected unit column stride")
    if ld < cols:
        if rows > 1:
            raise InvalidProblem(f"{name}: rows overlap")
        ld = cols
    return t.data_ptr(), ld


def _vector(t: Optional[torch.Tensor], dtype, elems: int, name: str, device: int) -> int:
    """Pointer of a contiguous vector of `dtype` with at least `elems` elements on `device`."""
    if t is None:
        raise InvalidProblem(f"{name} is required")
    if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous():
        raise InvalidProblem(f"{name}: expected a contiguous {dtype} device buffer, on the device of the others")
    if t.numel() < elems:
        raise BufferTooSmall(f"{name}: need {elems} elements, buffer holds {t.numel()}")
    return t.data_ptr()


def _call(device: int, stream, fn, *args) -> int:
    """fn(*args, stream) with the tensors' device as the current one; stream None is that device's current stream."""
    if stream is None:
        s = torch._C._cuda_getCurrentRawStream(device)
    else:
        s = stream if isinstance(stream, int) else stream.cuda_stream
    if torch._C._cuda_getDevice() == device:
        return fn(*args, s)
    with torch.cuda.device(device):
        return fn(*args, s)


# --------------------------------------------------------------------------- the cache
@dataclass(frozen=True)
class Kv4CacheDescriptor:
    """Geometry of one layer's cache.  The buffer is uint8 [num_pages, >= page_bytes] (its row pitch is the page stride)."""
    num_pages: int
    page_size: int
    heads_kv: int
    head_dim: int

    @property
    def page_bytes(self) -> int:
        if max(self.page_size, self.heads_kv, self.head_dim) >= 2**31:
            return 0  # not served
        return int(_lib.load().baracuda_kernels_kv4_page_bytes(self.page_size, self.heads_kv, self.head_dim))


def _cache(t: Optional[torch.Tensor], d: Kv4CacheDescriptor, page_bytes: int, device: int) -> tuple:
    """(pointer, page stride, pages, page size) of the cache buffer."""
    if t is None:
        raise InvalidProblem("cache is required")
    shape = t.shape
    if t.dtype is not torch.uint8 or t.get_device() != device or len(shape) != 2:
        raise InvalidProblem("cache: expected a uint8 matrix [num_pages, page_bytes] on the device of the others")
    if shape[0] < d.num_pages or shape[1] < page_bytes:
        raise BufferTooSmall(f"cache: need [{d.num_pages}, {page_bytes}] bytes, got {list(shape)}")
    stride, unit = t.stride()
    if unit != 1:
        raise InvalidProblem("cache: expected unit column stride")
    if stride < page_bytes:
        if d.num_pages > 1:
            raise InvalidProblem("cache: pages overlap")
        stride = page_bytes
    return t.data_ptr(), stride, d.num_pages, d.page_size


def _check_cache(d: Kv4CacheDescriptor) -> int:
    if d.num_pages < 0:
        raise InvalidProblem("negative dimension")
    if d.num_pages >= 2**31:
        raise InvalidProblem("dimension exceeds int32")
    return d.page_bytes


def _check_dims(*dims: int) -> None:
    if min(dims) < 0:
        raise InvalidProblem("negative dimension")
    if max(dims) >= 2**31:
        raise InvalidProblem("dimension exceeds int32")


# --------------------------------------------------------------------------- norms, rotation, append
@dataclass(frozen=True)
class QkNormRopeDescriptor:
    """`rot_dim` channels are rotated (default: all; 0: none), as halves or in neighbouring pairs (`interleaved`).
    `axis_of_pair` gives the position axis of each of the rot_dim / 2 pairs (None: one axis).  With `cache` the keys go to the
    4-bit cache, with the values beside them, instead of to `k_out`."""
    tokens: int
    heads_q: int
    heads_kv: int
    head_dim: int
    rot_dim: Optional[int] = None
    interleaved: bool = False
    axis_of_pair: Optional[Sequence[int]] = None
    eps: float = 1e-6
    cache: Optional[Kv4CacheDescriptor] = None


@dataclass
class QkNormRopeArgs:
    """bf16 q, k (and v); `cos_sin` float [max_pos, rot_dim] (cosines of the pairs, then sines); `positions` int32 [tokens] or
    [axes, tokens]; weights float [head_dim] or None for no norm; `slots` int64 [tokens], negative to leave a token out."""
    q: Optional[torch.Tensor]
    k: torch.Tensor
    q_out: Optional[torch.Tensor] = None
    cos_sin: Optional[torch.Tensor] = None
    positions: Optional[torch.Tensor] = None
    q_weight: Optional[torch.Tensor] = None
    k_weight: Optional[torch.Tensor] = None
    k_out: Optional[torch.Tensor] = None
    v: Optional[torch.Tensor] = None
    cache: Optional[torch.Tensor] = None
    slots: Optional[torch.Tensor] = None


class QkNormRopePlan:
    """RMS norm of every query and key head and the rotation by position, one pass, one launch; to bf16 or into the cache."""

    def __init__(self, desc: QkNormRopeDescriptor, rot_dim: int, axes: int, axis_of_pair, page_bytes: int):
        self.desc, self._rot, self._axes, self._axis_of_pair, self._page_bytes = desc, rot_dim, axes, axis_of_pair, page_bytes
        base = "baracuda_kernels_qk_norm_rope_" + ("kv4_append_" if desc.cache is not None else "") + "bf16_sm100a"
        self._fn = getattr(_lib.load(), base + "_run")

    @classmethod
    def select(cls, stream, desc: QkNormRopeDescriptor, pref: PlanPreference = PlanPreference()) -> "QkNormRopePlan":
        _check_backend(pref)
        rot = desc.head_dim if desc.rot_dim is None else desc.rot_dim
        _check_dims(desc.tokens, desc.heads_q, desc.heads_kv, desc.head_dim, rot)
        axes, table, page_bytes = 1, None, 0
        if desc.axis_of_pair is not None:
            given = [int(a) for a in desc.axis_of_pair]
            if len(given) != rot // 2 or any(a < 0 or a > 7 for a in given):
                raise InvalidProblem("axis_of_pair: expected rot_dim / 2 axis numbers from 0 to 7")
            axes = max(given, default=0) + 1
            table = (C.c_uint8 * max(1, len(given)))(*given)
        lib = _lib.load()
        if desc.cache is not None:
            _check_dims(desc.cache.page_size)
            if (desc.cache.heads_kv, desc.cache.head_dim) != (desc.heads_kv, desc.head_dim):
                raise InvalidProblem("the cache has other heads")
            status_to_result(lib.baracuda_kernels_qk_norm_rope_kv4_append_bf16_sm100a_can_implement(
                desc.tokens, desc.heads_q, desc.heads_kv, desc.head_dim, rot, axes, desc.cache.page_size), "QkNormRopePlan")
            page_bytes = _check_cache(desc.cache)
        else:
            status_to_result(lib.baracuda_kernels_qk_norm_rope_bf16_sm100a_can_implement(
                desc.tokens, desc.heads_q, desc.heads_kv, desc.head_dim, rot, axes), "QkNormRopePlan")
        return cls(desc, rot, axes, table, page_bytes)

    def workspace_size(self) -> int:
        return 0

    def run(self, stream, workspace: Optional[torch.Tensor], args: QkNormRopeArgs) -> None:
        d = self.desc
        t, hq, hkv, dim = d.tokens, d.heads_q, d.heads_kv, d.head_dim
        if t == 0:
            return
        dev = _device_of(args.k, "k")
        k, ldk = _matrix(args.k, t, hkv * dim, "k", dev)
        q, ldq, q_out, ldqo = None, 0, None, 0
        if hq:
            q, ldq = _matrix(args.q, t, hq * dim, "q", dev)
            q_out, ldqo = _matrix(args.q_out, t, hq * dim, "q_out", dev)
        wq = wk = table = positions = None
        if args.q_weight is not None:
            wq = _vector(args.q_weight, torch.float32, dim, "q_weight", dev)
        if args.k_weight is not None:
            wk = _vector(args.k_weight, torch.float32, dim, "k_weight", dev)
        max_pos = pos_stride = 0
        if self._rot:
            table = _vector(args.cos_sin, torch.float32, self._rot, "cos_sin", dev)
            shape = args.cos_sin.shape
            if len(shape) != 2 or shape[1] != self._rot:
                raise InvalidProblem(f"cos_sin: expected [max_pos, {self._rot}]")
            max_pos = min(shape[0], 2**31 - 1)  # positions are int32
            positions = _vector(args.positions, torch.int32, 1, "positions", dev)
            shape = args.positions.shape
            pos_stride = shape[-1] if shape else 0
            if len(shape) not in (1, 2):
                raise InvalidProblem("positions: expected [tokens] or [axes, tokens]")
            if pos_stride < t or (shape[0] if len(shape) == 2 else 1) < self._axes:
                raise BufferTooSmall(f"positions: need [{self._axes}, {t}]")
        if d.cache is None:
            k_out, ldko = _matrix(args.k_out, t, hkv * dim, "k_out", dev)
            st = _call(dev, stream, self._fn, t, hq, hkv, dim, q, ldq, k, ldk, wq, wk, d.eps, table, self._rot, max_pos, d.interleaved,
                       positions, pos_stride, self._axes, self._axis_of_pair, q_out, ldqo, k_out, ldko, None, 0)
        else:
            v, ldv = _matrix(args.v, t, hkv * dim, "v", dev)
            st = _call(dev, stream, self._fn, t, hq, hkv, dim, q, ldq, k, ldk, v, ldv, wq, wk, d.eps, table, self._rot, max_pos,
                       d.interleaved, positions, pos_stride, self._axes, self._axis_of_pair, q_out, ldqo,
                       *_cache(args.cache, d.cache, self._page_bytes, dev), _vector(args.slots, torch.int64, t, "slots", dev), None, 0)
        if st:
            status_to_result(st, "QkNormRopePlan")


@dataclass(frozen=True)
class Kv4AppendDescriptor:
    tokens: int
    cache: Kv4CacheDescriptor


@dataclass
class Kv4AppendArgs:
    """bf16 keys and values [tokens, heads_kv * head_dim], as the cache shall hold them."""
    k: torch.Tensor
    v: torch.Tensor
    cache: torch.Tensor
    slots: torch.Tensor


class Kv4AppendPlan:
    """Keys and values into the 4-bit cache, without norm or rotation (a cache filled from elsewhere, cross attention)."""

    _base = "baracuda_kernels_kv4_append_bf16_sm100a"

    def __init__(self, desc, page_bytes: int):
        self.desc, self._page_bytes = desc, page_bytes
        self._fn = getattr(_lib.load(), self._base + "_run")

    @classmethod
    def select(cls, stream, desc, pref: PlanPreference = PlanPreference()):
        _check_backend(pref)
        c = desc.cache
        _check_dims(desc.tokens, c.heads_kv, c.head_dim, c.page_size)
        status_to_result(getattr(_lib.load(), cls._base + "_can_implement")(desc.tokens, c.heads_kv, c.head_dim, c.page_size), cls.__name__)
        return cls(desc, _check_cache(c))

    def workspace_size(self) -> int:
        return 0

    def run(self, stream, workspace: Optional[torch.Tensor], args: Kv4AppendArgs) -> None:
        c, t = self.desc.cache, self.desc.tokens
        if t == 0:
            return
        dev, cols = _device_of(args.cache, "cache"), c.heads_kv * c.head_dim
        st = _call(dev, stream, self._fn, t, c.heads_kv, c.head_dim, *_matrix(args.k, t, cols, "k", dev), *_matrix(args.v, t, cols, "v", dev),
                   *_cache(args.cache, c, self._page_bytes, dev), _vector(args.slots, torch.int64, t, "slots", dev), None, 0)
        if st:
            status_to_result(st, "Kv4AppendPlan")


@dataclass(frozen=True)
class Kv4ReadDescriptor:
    tokens: int
    cache: Kv4CacheDescriptor


@dataclass
class Kv4ReadArgs:
    cache: torch.Tensor
    slots: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor


class Kv4ReadPlan(Kv4AppendPlan):
    """The tokens at `slots` as bf16 keys and values (a prefix handed to another engine or stored elsewhere)."""

    _base = "baracuda_kernels_kv4_read_bf16_sm100a"

    def run(self, stream, workspace: Optional[torch.Tensor], args: Kv4ReadArgs) -> None:
        c, t = self.desc.cache, self.desc.tokens
        if t == 0:
            return
        dev, cols = _device_of(args.cache, "cache"), c.heads_kv * c.head_dim
        st = _call(dev, stream, self._fn, t, c.heads_kv, c.head_dim, *_cache(args.cache, c, self._page_bytes, dev),
                   _vector(args.slots, torch.int64, t, "slots", dev), *_matrix(args.k, t, cols, "k", dev), *_matrix(args.v, t, cols, "v", dev),
                   None, 0)
        if st:
            status_to_result(st, "Kv4ReadPlan")


# --------------------------------------------------------------------------- attention
@dataclass(frozen=True)
class Kv4AttentionDescriptor:
    """`max_q` and `max_kv` bound the rows and cached tokens of any sequence (what a captured graph may meet), and the launch is cut
    for them: prompts and single tokens are better served by a call each.  `window` > 0 lets a row see that many keys back, its own
    included; `scale` defaults to head_dim ** -0.5."""
    batch: int
    max_q: int
    max_kv: int
    heads_q: int
    cache: Kv4CacheDescriptor
    causal: bool = True
    window: int = 0
    scale: Optional[float] = None


@dataclass
class Kv4AttentionArgs:
    """q, out bf16 [total_q, heads_q * head_dim]; cu_q int32 [batch + 1]; kv_lens int32 [batch]; page_table int32
    [batch, >= ceil(max_kv / page_size)]; lse float [total_q, heads_q] or None."""
    q: torch.Tensor
    cu_q: torch.Tensor
    kv_lens: torch.Tensor
    page_table: torch.Tensor
    cache: torch.Tensor
    out: torch.Tensor
    lse: Optional[torch.Tensor] = None


class Kv4AttentionPlan:
    """Attention of ragged query rows over the 4-bit cache: decode steps, drafted tokens, prompts."""

    _base = "baracuda_kernels_attention_kv4_bf16_sm100a"

    def __init__(self, desc: Kv4AttentionDescriptor, scale: float, page_bytes: int):
        self.desc, self._scale, self._page_bytes = desc, scale, page_bytes
        lib = _lib.load()
        c = desc.cache
        self._fn = getattr(lib, self._base + "_run")
        self._workspace = int(getattr(lib, self._base + "_workspace_size")(desc.batch, desc.max_q, desc.max_kv, desc.heads_q,
                                                                           c.heads_kv, c.head_dim))

    @classmethod
    def select(cls, stream, desc: Kv4AttentionDescriptor, pref: PlanPreference = PlanPreference()) -> "Kv4AttentionPlan":
        _check_backend(pref)
        c = desc.cache
        _check_dims(desc.batch, desc.max_q, desc.max_kv, desc.heads_q, c.heads_kv, c.head_dim, c.page_size, desc.window)
        status_to_result(getattr(_lib.load(), cls._base + "_can_implement")(
            desc.batch, desc.max_q, desc.max_kv, desc.heads_q, c.heads_kv, c.head_dim, c.page_size), cls.__name__)
        scale = c.head_dim ** -0.5 if desc.scale is None else float(desc.scale)
        if not abs(scale) <= torch.finfo(torch.float32).max:
            raise InvalidProblem("scale must be finite, in 32 bits too")
        plan = cls(desc, scale, _check_cache(c))
        if plan.workspace_size() > pref.max_workspace_bytes:
            raise Unsupported("workspace budget too small for this shape")
        return plan

    def workspace_size(self) -> int:
        return self._workspace

    def run(self, stream, workspace: Optional[torch.Tensor], args: Kv4AttentionArgs) -> None:
        d = self.desc
        c = d.cache
        if d.batch == 0 or d.max_q == 0:
            return
        dev, cols = _device_of(args.q, "q"), d.heads_q * c.head_dim
        total = args.q.shape[0] if args.q.dim() else 0
        if total == 0:
            return
        q, ldq = _matrix(args.q, total, cols, "q", dev)
        out, ldo = _matrix(args.out, total, cols, "out", dev)
        lse = None if args.lse is None else _vector(args.lse, torch.float32, total * d.heads_q, "lse", dev)
        table = args.page_table
        if table is None or table.dtype is not torch.int32 or table.get_device() != dev:
            raise InvalidProblem("page_table: expected an int32 matrix [batch, pages] on the device of the others")
        shape = table.shape
        if len(shape) != 2 or shape[0] < d.batch or shape[1] * c.page_size < d.max_kv:
            raise BufferTooSmall(f"page_table: need [{d.batch}, {-(-d.max_kv // c.page_size)}], got {list(shape)}")
        ld_table, unit = table.stride()
        if shape[1] > 1 and unit != 1:
            raise InvalidProblem("page_table: expected unit column stride")
        if ld_table < shape[1]:
            if d.batch > 1:
                raise InvalidProblem("page_table: rows overlap")
            ld_table = shape[1]
        ws, ws_bytes = None, 0
        if self._workspace:
            if workspace is not None:
                ws, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
                if workspace.get_device() != dev or not workspace.is_contiguous():
                    raise InvalidProblem("workspace: expected a contiguous device buffer, on the device of the others")
            if self._workspace > ws_bytes:
                raise WorkspaceTooSmall(self._workspace, ws_bytes)
        st = _call(dev, stream, self._fn, d.batch, total, d.max_q, d.max_kv, d.heads_q, c.heads_kv, c.head_dim, q, ldq,
                   _vector(args.cu_q, torch.int32, d.batch + 1, "cu_q", dev), *_cache(args.cache, c, self._page_bytes, dev), table.data_ptr(),
                   ld_table, _vector(args.kv_lens, torch.int32, d.batch, "kv_lens", dev), self._scale, d.causal, d.window, out, ldo, lse, ws,
                   ws_bytes)
        if st:
            status_to_result(st, "Kv4AttentionPlan")
