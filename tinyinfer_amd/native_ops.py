"""Torch-facing ctypes binding of the v2 kernel ABI (libtinyinfer_backend.so).

The public surface is the one reference llm/native_ops.py:33-210 gives its
callers: ``NativeOps`` with ``gemm``, ``gemm_int8``, ``legacy_gemm``,
``layernorm``, ``gelu_new``, ``softmax`` and ``attention``; the module constant
``GEMM_CATALOG`` (reference :14-16) that the library's catalog JSON must equal;
and the exception contract -- ``TypeError`` for an operand that is not a
contiguous device tensor of the right dtype, ``ValueError`` for a bad rank,
extent, device, integer argument or a tensor that requires grad,
``RuntimeError`` carrying ``ti_v2_last_error()`` for a nonzero native status.
Beyond it: an int8 KV cache (``kv_cache_int8``, ``kv_append_int8``,
``kv_read_int8``), attention over it for single tokens and prompts
(``attention_int8kv``, ``attention_shared_prefix``) and ``sample``, one token per
row of logits; rotary positions (``rotary``, ``rotate``), a paged fp16 KV cache
(``kv_cache_paged``, ``kv_append_paged`` with the rotation on the way,
``kv_read_paged``), attention over it (``attention_paged``) and ``logprobs``, the log
probabilities of given tokens with their row's entropy and likeliest tokens.

How it is built here: every native symbol is described by a string of
parameter codes (``_ABI``); each call goes through a ``_Call`` that validates
the operands in argument order, allocates outputs on the operands' device,
records the caller's tensors on the current torch stream (the allocator must not
recycle them while the queued kernels run; outputs and metadata come from that
stream's own pool), and appends that stream and the device index as the ABI's
last two arguments.  There is no CPU path: the
library must be built, and the operands must already live on the GPU.
"""
from __future__ import annotations

import ctypes
import itertools
import json
import math
import sys
import warnings
from array import array
from contextlib import nullcontext
from pathlib import Path

from . import BACKEND_LIB, require

INT32_MAX = 2**31 - 1
INT64_MAX = 2**63 - 1
_FLOAT_MAX = sys.float_info.max

# The 12 GEMM configurations the library must report, in order (the reference
# catalog, kernels/src/cuda/tc/catalog.cuh:8-15): three CUDA tile hints, one or
# two stages, fused bias epilogue for ids 0-5, a caller FP32 workspace for 6-11.
_TILE_HINTS = ((32, 32, 16, 4), (64, 32, 32, 8), (64, 64, 32, 8))
GEMM_CATALOG = tuple(
    {"id": cid, "tile": _TILE_HINTS[cid % 3],
     "stages": 2 if (cid % 6) < 3 else 1,
     "epilogue": "fused" if cid < 6 else "separate"}
    for cid in range(12))

# Parameter codes of each entry point, before the implicit (stream, device)
# trailer: p = pointer, i = int, f = float, q = int64.
_ABI = {
    "ti_v2_gemm_f16": "ppppiiiii",
    "ti_v2_gemm_i8": "pppppiiiii",
    "ti_v2_gemm_ex_f16": "pppppiiiii",
    "ti_v2_gemm_ex_i8": "ppppppiiiii",
    "ti_v2_legacy_gemm_f32": "pppiii",
    "ti_v2_attention_f16": "pppppppiiiiiii",
    "ti_v2_layernorm_f16": "ppppiif",
    "ti_v2_gelu_new_f16": "ppq",
    "ti_v2_softmax_f16": "ppii",
    "ti_amd_kv_append_i8": "ppppppii",
    "ti_amd_kv_read_i8": "ppppppii",
    "ti_amd_attention_i8kv": "ppppppppqiiiiiii",
    "ti_amd_sample": "pippppp" "fiff" "ppii",
    "ti_amd_rotate": "pqqqppipiifiiii",
    "ti_amd_kv_append_paged": "ppqqqpqqqpqqqp" "pippp" "iifiii",
    "ti_amd_kv_read_paged": "ppppippii",
    "ti_amd_attention_paged": "ppppipppp" "qiiiii",
    "ti_amd_logprobs": "pipppppiiii",
}
_CTYPE = {"p": ctypes.c_void_p, "i": ctypes.c_int, "f": ctypes.c_float, "q": ctypes.c_int64}
_TRAILER = [ctypes.c_size_t, ctypes.c_int]   # hipStream_t as uintptr_t, device ordinal


def _count(value, name, low=1, high=INT32_MAX):
    """An exact int (bool excluded) in [low, high], else ValueError."""
    if type(value) is not int or value < low or value > high:
        raise ValueError(f"{name} must be an integer in [{low}, {high}]")
    return value


def _per_request(value, batch, default, upper, name):
    """Host metadata for each of `batch` requests: None (every request gets
    `default`), a single int for all, or a sequence of `batch` ints in [0, upper]."""
    if value is None:
        return [default] * batch
    seq = [value] * batch if type(value) is int else list(value)
    if len(seq) != batch:
        raise ValueError(f"{name} must hold {batch} entries, got {len(seq)}")
    if set(map(type, seq)) != {int} or min(seq) < 0 or max(seq) > upper:
        for item in seq:
            _count(item, name, 0, upper)
    return seq


class _Call:
    """One native call being assembled: operands are checked and their
    pointers appended in the ABI's argument order.

    A small call's time is this Python code (a GEMV runs 5 us on the GPU), so an
    operand that passes every check is accepted by one native call (csrc/operands.cpp)
    and only a refused one goes through the ordered checks that name the reason; outputs
    come from the calling stream's own pool and need no record_stream; the
    device is switched only when it is not current.  ``gemm_int8`` at M = 1,
    768 -> 2304, call after call: 15.6 us with every check in turn, 7.4 now."""

    __slots__ = ("ops", "symbol", "args", "held", "made", "like", "index", "over", "turned")

    def __init__(self, ops, symbol):
        self.ops, self.symbol = ops, symbol
        self.args = []
        self.held, self.made = [], []   # the caller's tensors, and this call's own
        self.like = None                # a tensor where the call's operands are
        self.index = -2                 # its GPU; -2: none yet
        self.over = None                # the cache it works on
        self.turned = None              # the rotary positions it turns rows by

    @property
    def device(self):
        return None if self.like is None else self.like.device

    def operand(self, x, dtype, name, rank=None, shape=None):
        # (At most INT32_MAX elements: then every extent and the byte count fit.)
        at = self.ops.operands.operand(x, dtype, self.index, -1 if rank is None else rank, shape)
        if at is None:
            self._checked(x, dtype, name, rank, shape)
            at = x.data_ptr()
        if self.like is None:
            self.like = x
            self.index = x.get_device()
        self.held.append(x)
        self.args.append(at)
        return x

    def _checked(self, x, dtype, name, rank, shape, strided=False):
        """The operand checks one by one, each with its own exception (strided: the last axis
        alone must be contiguous)."""
        torch = self.ops.torch
        if not isinstance(x, torch.Tensor) or x.device.type != "cuda":
            raise TypeError(f"{name}: a GPU (torch 'cuda' device) tensor is required")
        if x.dtype != dtype:
            raise TypeError(f"{name}: dtype {x.dtype} given, {dtype} required")
        if not x.is_contiguous() and not strided:
            raise TypeError(f"{name}: contiguous row-major storage required")
        if strided and x.dim() and x.shape[-1] > 1 and x.stride(-1) != 1:
            raise TypeError(f"{name}: a last axis of contiguous values required")
        if x.requires_grad:
            raise ValueError(f"{name}: tensors that require grad are not accepted (inference only)")
        if rank is not None and x.dim() != rank:
            raise ValueError(f"{name}: rank {rank} required, got {x.dim()}")
        if x.dim() == 0 or x.numel() == 0:
            raise ValueError(f"{name}: an empty or zero-rank tensor is not accepted")
        for axis, extent in enumerate(x.shape):
            _count(extent, f"{name}.shape[{axis}]")
        if x.numel() * x.element_size() > INT64_MAX:
            raise ValueError(f"{name}: byte extent beyond signed 64-bit indexing")
        if self.device is not None and x.device != self.device:
            raise ValueError(f"{name}: on {x.device}, the call's operands are on {self.device}")
        if shape is not None and tuple(x.shape) != tuple(shape):
            raise ValueError(f"{name}: shape {tuple(shape)} required, got {tuple(x.shape)}")

    def optional(self, x, dtype, name, shape):
        if x is None:
            self.args.append(None)
            return None
        return self.operand(x, dtype, name, shape=shape)

    def rows(self, x, name, shape):
        """fp16 rows [B,H,Q,D] of the given shape (None: any) in any layout whose dims
        are contiguous, a slice of a projection for one: pointer and three strides.
        Returns its shape."""
        half = self.ops.torch.float16
        at = self.ops.operands.rows(x, half, self.index, shape)
        if at is None:
            self._checked(x, half, name, 4, shape, strided=True)
            at = (x.data_ptr(), *x.stride()[:3])
        if self.like is None:
            self.like = x
            self.index = x.get_device()
        self.held.append(x)
        self.args += at
        return x.shape

    def output(self, shape, dtype):
        y = self.ops.operands.empty_as(shape, dtype, self.like)
        self.made.append(y)
        self.args.append(y.data_ptr())
        return y

    def output_like(self, x):
        y = self.ops.operands.empty(x.shape, x)
        self.made.append(y)
        self.args.append(y.data_ptr())
        return y

    def workspace(self, shape, needed):
        if not needed:
            self.args.append(None)
            return None
        return self.output(shape, self.ops.torch.float32)

    def metadata(self, *lists):
        """Equal-length int lists as device int32 arrays, in one copy from pinned
        memory that the stream orders before the call (a copy from pageable
        memory would wait for everything queued on the stream before it; three
        such copies made a 32-request decode call 73 us, this one 27)."""
        torch = self.ops.torch
        with torch.cuda.device(self.device) if torch.cuda.current_device() != self.device.index else nullcontext():
            capturing = torch.cuda.is_current_stream_capturing()
        if capturing:
            raise RuntimeError(f"{self.symbol}: host metadata cannot be captured into a graph")
        flat = array("i", itertools.chain(*lists))
        host = torch.empty(len(flat), dtype=torch.int32, pin_memory=True)
        host.copy_(torch.frombuffer(flat, dtype=torch.int32))
        held = host.to(self.device, non_blocking=True)
        self.made.append(held)
        at = held.data_ptr()
        self.args.extend(at + 4 * len(lists[0]) * i for i in range(len(lists)))

    def cache(self, cache, kind=None):
        if type(cache) is not (kind or Int8KVCache):
            raise TypeError("cache: an Int8KVCache (NativeOps.kv_cache_int8) is required" if kind is None else
                            "cache: a PagedKVCache (NativeOps.kv_cache_paged) is required")
        self.like = cache.buffer
        self.index = cache.buffer.get_device()
        self.over = cache
        self.args.append(cache._at)

    def page_table(self, table, batch):
        """int32 [B,W] on the call's device, W pages to a request."""
        self.operand(table, self.ops.torch.int32, "page_table", rank=2)
        rows, width = table.shape
        if rows != batch:
            raise ValueError(f"page_table: a row for each of {batch} requests required, got {rows}")
        self.args.append(width)
        return width

    def turn(self, rotary):
        """The frequencies' pointer, the turned dims, the layout and the factor."""
        if rotary is None:
            self.args.extend((None, 0, 0, 1.0))
            return
        if rotary.turns.get_device() != self.index:
            raise ValueError(f"rotary: on {rotary.turns.device}, the call's operands are on {self.device}")
        self.turned = rotary
        self.args.extend((rotary._at, rotary.rotated, int(rotary.interleaved), rotary.amplitude))

    def per_request(self, batch, *items):
        """One int per request, each item (value, upper, name): int32 [batch] tensors on
        the call's device, whose values the kernels bound, or host ints or sequences
        of them in [0, upper], checked here.  None stays null."""
        torch, host, where = self.ops.torch, [], []
        for value, upper, name in items:
            if value is None:
                self.args.append(None)
            elif isinstance(value, self.ops.tensor_type):
                self.operand(value, torch.int32, name, shape=(batch,))
            else:
                host.append(_per_request(value, batch, 0, upper, name))
                where.append(len(self.args))
                self.args.append(None)
        if host:
            at = len(self.args)
            self.metadata(*host)
            for i, pointer in zip(where, self.args[at:]):
                self.args[i] = pointer
            del self.args[at:]

    def scalars(self, *values):
        self.args.extend(values)

    def run(self):
        ops, index = self.ops, self.index
        cuda = ops.torch.cuda
        # (The current stream's handle costs a tenth of making its Stream object, whose number
        # record_stream wants and which stays the same for a handle.)
        handle = ops.stream_handle(index)
        stream = ops.streams.get((index, handle))
        if stream is None:
            stream = cuda.current_stream(index)
            stream = ops.streams[index, handle] = stream if type(ops.operands) is _PlainOperands else stream.stream_id
        ops.operands.record(self.held, stream, index)
        # (The allocator keeps a stream with a block until the block is freed: once does.)
        if self.over is not None and handle not in self.over._streams:
            ops.operands.record([self.over.buffer], stream, index)
            self.over._streams.add(handle)
        if self.turned is not None and handle not in self.turned._streams:
            ops.operands.record([self.turned.turns], stream, index)
            self.turned._streams.add(handle)
        if ops.current_device() == index:
            status = getattr(ops.lib, self.symbol)(*self.args, handle, index)
        else:
            with cuda.device(self.device):
                status = getattr(ops.lib, self.symbol)(*self.args, handle, index)
        if status != 0:
            detail = ops.lib.ti_v2_last_error().decode("utf-8", errors="replace")
            raise RuntimeError(f"{self.symbol} failed ({status}): {detail}")


class _KvI8(ctypes.Structure):
    """ti_amd_kv_i8."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scales", ctypes.c_void_p),
                ("v_scales", ctypes.c_void_p), ("slots", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("capacity", ctypes.c_int32), ("head_dim", ctypes.c_int32)]


class Int8KVCache:
    """An int8 KV cache of `slots` requests, made by ``NativeOps.kv_cache_int8``.

    One zeroed buffer holds K's and V's bytes and their fp32 scales (one per
    token and head), in the order include/tinyinfer_amd_ext.h describes; rows go in
    through ``kv_append_int8`` and come back through ``kv_read_int8``.  `capacity`
    is the requested one rounded up to a multiple of 64.  The cache keeps no
    lengths: every call names the slots, positions and lengths it means."""

    __slots__ = ("slots", "kv_heads", "capacity", "head_dim", "buffer", "_native", "_at", "_workspace", "_streams")

    def __init__(self, torch, slots, kv_heads, capacity, head_dim, device):
        capacity = (capacity + 63) // 64 * 64
        tokens = slots * kv_heads * capacity
        buffer = torch.zeros(tokens * (2 * head_dim + 8), dtype=torch.uint8, device=device)
        at = buffer.data_ptr()
        native = _KvI8(at, at + tokens * head_dim, at + 2 * tokens * head_dim, at + 2 * tokens * head_dim + 4 * tokens,
                       slots, kv_heads, capacity, head_dim)
        # _workspace: bytes an attention call needs, by its shape; _streams: those that
        # the allocator has been told of.
        for name, value in (("slots", slots), ("kv_heads", kv_heads), ("capacity", capacity), ("head_dim", head_dim),
                            ("buffer", buffer), ("_native", native), ("_at", ctypes.addressof(native)),
                            ("_workspace", {}), ("_streams", set())):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"{name}: a cache's buffer and extents stay as they were made")

    @property
    def device(self):
        return self.buffer.device


class _KvPaged(ctypes.Structure):
    """ti_amd_kv_paged."""
    _fields_ = [("pages", ctypes.c_void_p), ("page_count", ctypes.c_int32), ("kv_heads", ctypes.c_int32),
                ("page_size", ctypes.c_int32), ("head_dim", ctypes.c_int32)]


class PagedKVCache:
    """A paged fp16 KV cache, made by ``NativeOps.kv_cache_paged``.

    ``buffer`` [pages, kv_heads * 2 * page_size * head_dim] is zeroed; a page's inner order
    is the kernels' own, so rows go in through ``kv_append_paged`` and come back through
    ``kv_read_paged``, but a page is one row of it: ``cache.buffer[a] = cache.buffer[b]``
    copies page b to page a.  Which pages a request's tokens lie on is the caller's
    table: token t of request b on page ``table[b, t // page_size]``; a number outside the
    cache, -1 for one, stands for no page."""

    __slots__ = ("pages", "kv_heads", "page_size", "head_dim", "buffer", "_native", "_at", "_workspace", "_streams")

    def __init__(self, torch, pages, kv_heads, page_size, head_dim, device):
        buffer = torch.zeros((pages, kv_heads * 2 * page_size * head_dim), dtype=torch.float16, device=device)
        native = _KvPaged(buffer.data_ptr(), pages, kv_heads, page_size, head_dim)
        for name, value in (("pages", pages), ("kv_heads", kv_heads), ("page_size", page_size), ("head_dim", head_dim),
                            ("buffer", buffer), ("_native", native), ("_at", ctypes.addressof(native)),
                            ("_workspace", {}), ("_streams", set())):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"{name}: a cache's buffer and extents stay as they were made")

    @property
    def device(self):
        return self.buffer.device


class Rotary:
    """Rotary positions, made by ``NativeOps.rotary``: the first `rotated` dims of a row are
    turned, pair i by ``frequencies[i]`` radians a position; turned values are multiplied by
    `amplitude`.  ``turns`` holds the frequencies on the device, as 2^64 (f / 2 pi mod 1)."""

    __slots__ = ("rotated", "interleaved", "amplitude", "frequencies", "turns", "_at", "_streams")

    def __init__(self, torch, frequencies, interleaved, amplitude, device):
        whole = [round(math.fmod(f / (2 * math.pi), 1.0) * 2.0 ** 64) % 2 ** 64 for f in frequencies]
        turns = torch.tensor([n - 2 ** 64 if n >= 2 ** 63 else n for n in whole], dtype=torch.int64, device=device)
        for name, value in (("rotated", 2 * len(frequencies)), ("interleaved", interleaved), ("amplitude", float(amplitude)),
                            ("frequencies", tuple(frequencies)), ("turns", turns), ("_at", turns.data_ptr()),
                            ("_streams", set())):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError(f"{name}: rotary positions stay as they were made")


def _number(value, name, low=-math.inf, above=False):
    """A finite number >= low (> low if above), else ValueError."""
    # (An int beyond every float is not finite either.)
    if type(value) not in (int, float) or not abs(value) <= _FLOAT_MAX or value < low or (above and value == low):
        raise ValueError(f"{name} must be a finite number {'above' if above else 'of at least'} {low}")
    return value


class _PlainOperands:
    """csrc/operands.cpp in Python, for a torch that it was not compiled for."""

    def __init__(self, torch):
        self.torch = torch

    def _accepts(self, x, dtype, index, shape):
        return (isinstance(x, self.torch.Tensor) and x.dtype == dtype and x.is_cuda and index in (-2, x.get_device())
                and not x.requires_grad and 0 < x.numel() <= INT32_MAX and (shape is None or x.shape == shape))

    def operand(self, x, dtype, index, rank, shape):
        if self._accepts(x, dtype, index, shape) and x.is_contiguous() and x.dim() and rank in (x.dim(), -1):
            return x.data_ptr()
        return None

    def rows(self, x, dtype, index, shape):
        if self._accepts(x, dtype, index, shape) and x.dim() == 4 and 1 in (x.stride(3), x.shape[3]):
            return (x.data_ptr(), *x.stride()[:3])
        return None

    def empty(self, shape, like):
        return self.empty_as(shape, like.dtype, like)

    def empty_as(self, shape, dtype, like):
        return self.torch.empty(shape, dtype=dtype, device=like.device)

    def record(self, tensors, stream, index):
        for x in tensors:
            x.record_stream(stream)  # (a Stream object here)


def _operand_checks(torch):
    """csrc/operands.cpp if it is there and of this torch, else the same in Python."""
    try:
        from . import _operands  # (after torch, whose libraries it uses)
        if _operands.torch_version == torch.__version__:
            return _operands
        found = f"compiled for torch {_operands.torch_version}"
    except ImportError as e:
        found = f"not importable ({e})"
    warnings.warn(f"tinyinfer_amd._operands is {found}: calls are checked in Python, some microseconds slower each, under torch "
                  f"{torch.__version__}; python -m tinyinfer_amd.build compiles it", RuntimeWarning, stacklevel=3)
    return _PlainOperands(torch)


class NativeOps:
    """Inference-only device ops over the v2 ABI; operands are torch GPU tensors,
    work is queued on the current torch stream of their device."""

    def __init__(self, library_path=None):
        import torch
        self.torch, self.tensor_type, self.operands = torch, torch.Tensor, _operand_checks(torch)
        # torch's own short ways to both (operands are on a GPU: it is initialised), which
        # are not part of its interface and missing in a torch without GPU support.
        self.stream_handle = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        self.current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
        self.streams = {}
        where = require(BACKEND_LIB) if library_path is None else library_path
        self.library_path = str(Path(where).expanduser().resolve(strict=True))
        self.lib = ctypes.CDLL(self.library_path)
        self._declare("ti_v2_abi_version", [], ctypes.c_int)
        self._declare("ti_v2_last_error", [], ctypes.c_char_p)
        self._declare("ti_v2_gemm_catalog_json", [], ctypes.c_char_p)
        for symbol, codes in _ABI.items():
            self._declare(symbol, [_CTYPE[c] for c in codes] + _TRAILER, ctypes.c_int)
        if self.lib.ti_v2_abi_version() != 2:
            raise RuntimeError("native v2 ABI version mismatch: version 2 required")
        self._declare("ti_amd_attention_i8kv_workspace", [ctypes.c_void_p] + [ctypes.c_int] * 5, ctypes.c_int64)
        self._declare("ti_amd_attention_paged_workspace", [ctypes.c_void_p] + [ctypes.c_int] * 5, ctypes.c_int64)
        self.catalog = json.loads(self.lib.ti_v2_gemm_catalog_json())
        listed = tuple({**entry, "tile": tuple(entry["tile"])} for entry in self.catalog["configs"])
        if listed != GEMM_CATALOG:
            raise RuntimeError("native GEMM catalog differs from the wrapper's GEMM_CATALOG")

    def _declare(self, symbol, argtypes, restype):
        fn = getattr(self.lib, symbol)
        fn.argtypes, fn.restype = argtypes, restype

    # -- GEMMs --------------------------------------------------------------
    def _linear(self, symbol, a, weight, weight_dtype, scales, bias, config, output_dtype):
        torch = self.torch
        call = _Call(self, symbol)
        call.operand(a, torch.float16, "a", rank=2)
        call.operand(weight, weight_dtype, "b", rank=2)
        if scales is not None:
            call.operand(scales, torch.float32, "scales", rank=1)
            if scales.shape[0] != weight.shape[1]:
                raise ValueError("scales must have shape [N], one scale per output column")
        m, k = a.shape
        if weight.shape[0] != k:
            raise ValueError(f"a is [{m}, {k}] but b has {weight.shape[0]} rows")
        n = weight.shape[1]
        if type(config) is not int or config not in range(len(GEMM_CATALOG)):
            raise ValueError(f"GEMM config must be one of the catalog ids 0..{len(GEMM_CATALOG) - 1}")
        only = self.catalog.get("only_config", -1)
        if only not in (-1, config):
            raise ValueError(f"this build compiles only GEMM config {only}")
        rows_per_tile = GEMM_CATALOG[config]["tile"][0]
        if (m + rows_per_tile - 1) // rows_per_tile > 65535:
            raise ValueError("M needs more than 65535 row tiles")
        call.optional(bias, torch.float16, "bias", shape=(n,))
        out_dtype = torch.float16 if output_dtype is None else output_dtype
        if out_dtype not in (torch.float16, torch.float32):
            raise TypeError("output_dtype must be torch.float16 or torch.float32")
        y = call.output((m, n), out_dtype)
        call.workspace((m, n), GEMM_CATALOG[config]["epilogue"] == "separate")
        call.scalars(m, n, k, 1 if out_dtype == torch.float32 else 0, config)
        call.run()
        return y

    def gemm(self, a, b, *, bias=None, config=0, output_dtype=None):
        """y = a[M,K] @ b[K,N] (+ bias), fp16 weights, fp32 accumulation."""
        return self._linear("ti_v2_gemm_ex_f16", a, b, self.torch.float16, None, bias, config, output_dtype)

    def gemm_int8(self, a, b, scales, *, bias=None, config=0, output_dtype=None):
        """W8A16: b int8 [K,N] with one fp32 scale per output column."""
        if scales is None:
            raise TypeError("scales: a GPU (torch 'cuda' device) tensor is required")
        return self._linear("ti_v2_gemm_ex_i8", a, b, self.torch.int8, scales, bias, config, output_dtype)

    def legacy_gemm(self, a, b):
        """FP32 y = a @ b through ti_v2_legacy_gemm_f32."""
        torch = self.torch
        call = _Call(self, "ti_v2_legacy_gemm_f32")
        call.operand(a, torch.float32, "a", rank=2)
        call.operand(b, torch.float32, "b", rank=2)
        (m, k), n = a.shape, b.shape[1]
        if b.shape[0] != k or (m + 63) // 64 > 65535:
            raise ValueError(f"FP32 GEMM: a [{m}, {k}] and b {list(b.shape)} do not multiply within the grid limit")
        y = call.output((m, n), torch.float32)
        call.scalars(m, n, k)
        call.run()
        return y

    # -- row ops -------------------------------------------------------------
    def _rows(self, x):
        cols = x.shape[-1]
        return _count(x.numel() // cols, "rows"), cols

    def layernorm(self, x, gamma, beta, *, eps=1e-5):
        """fp16 LayerNorm over the last axis, gamma/beta fp16 [cols]."""
        torch = self.torch
        call = _Call(self, "ti_v2_layernorm_f16")
        call.operand(x, torch.float16, "x")
        rows, cols = self._rows(x)
        call.operand(gamma, torch.float16, "gamma", rank=1)
        call.operand(beta, torch.float16, "beta", rank=1)
        if gamma.shape[0] != cols or beta.shape[0] != cols:
            raise ValueError(f"gamma and beta must have shape [{cols}]")
        if not (isinstance(eps, (int, float)) and math.isfinite(eps) and eps > 0):
            raise ValueError("eps must be finite and positive")
        y = call.output(tuple(x.shape), torch.float16)
        call.scalars(rows, cols, float(eps))
        call.run()
        return y

    def gelu_new(self, x):
        """fp16 tanh-approximation GELU, elementwise."""
        call = _Call(self, "ti_v2_gelu_new_f16")
        call.operand(x, self.torch.float16, "x")
        y = call.output(tuple(x.shape), self.torch.float16)
        call.scalars(x.numel())
        call.run()
        return y

    def softmax(self, x):
        """fp16 softmax over the last axis."""
        call = _Call(self, "ti_v2_softmax_f16")
        call.operand(x, self.torch.float16, "x")
        rows, cols = self._rows(x)
        y = call.output(tuple(x.shape), self.torch.float16)
        call.scalars(rows, cols)
        call.run()
        return y

    # -- attention -------------------------------------------------------------
    def attention(self, q, k, v, *, q_lengths=None, kv_lengths=None, query_offsets=None,
                  causal=True, config=0):
        """q [B,H,Q,D], k/v [B,H,K,D] fp16, D in {64, 128}; per-request query
        and key counts and absolute query offsets for the causal mask."""
        torch = self.torch
        call = _Call(self, "ti_v2_attention_f16")
        call.operand(q, torch.float16, "q", rank=4)
        batch, heads, nq, dim = q.shape
        call.operand(k, torch.float16, "k", rank=4)
        call.operand(v, torch.float16, "v", rank=4)
        nk = k.shape[2]
        if (tuple(v.shape) != tuple(k.shape) or tuple(k.shape[:2]) != (batch, heads)
                or k.shape[3] != dim or dim not in (64, 128)):
            raise ValueError("attention takes q [B,H,Q,D] and k, v [B,H,K,D] with D 64 or 128")
        if batch > 65535 or heads > 65535:
            raise ValueError("batch and heads must each be at most 65535")
        if type(causal) is not bool or type(config) is not int or config not in (0, 1):
            raise ValueError("causal must be a bool and config 0 or 1")
        meta = (_per_request(q_lengths, batch, nq, nq, "q_lengths"),
                _per_request(kv_lengths, batch, nk, nk, "kv_lengths"),
                _per_request(query_offsets, batch, 0, INT32_MAX - nq, "query_offsets"))
        y = call.output(tuple(q.shape), torch.float16)
        call.metadata(*meta)
        call.scalars(batch, heads, nq, nk, dim, int(causal), config)
        call.run()
        return y

    # -- int8 KV cache ---------------------------------------------------------
    def kv_cache_int8(self, slots, kv_heads, capacity, head_dim, *, device=None):
        """A zeroed cache for `slots` requests of up to `capacity` tokens (rounded up
        to a multiple of 64), `kv_heads` key heads of 64 or 128 dims."""
        torch = self.torch
        _count(slots, "slots")
        _count(kv_heads, "kv_heads", high=65535)
        _count(capacity, "capacity", high=INT32_MAX - 63)
        if type(head_dim) is not int or head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        where = torch.device("cuda" if device is None else device)
        if where.type != "cuda":
            raise TypeError("device: a GPU (torch 'cuda' device) is required")
        return Int8KVCache(torch, slots, kv_heads, capacity, head_dim, where)

    def kv_append_int8(self, cache, k, v, slots, positions, *, lengths=None):
        """Quantise k, v fp16 [B,G,Q,D] into the cache as they are: row i < lengths[b]
        (None: Q) becomes token positions[b] + i of slots[b].

        slots, positions and lengths are int32 [B] tensors, or host ints (one for
        all, or B of them).  Host values must lie inside the cache; rows that device
        values put outside it are not written.  Where two requests write the same
        token, the later request's row stays."""
        torch = self.torch
        call = _Call(self, "ti_amd_kv_append_i8")
        call.cache(cache)
        call.operand(k, torch.float16, "k", rank=4)
        batch, heads, rows, dim = k.shape
        if heads != cache.kv_heads or dim != cache.head_dim:
            raise ValueError(f"k must be [B, {cache.kv_heads}, Q, {cache.head_dim}], got {list(k.shape)}")
        call.operand(v, torch.float16, "v", shape=k.shape)
        self._batch_rows(batch, slots, positions, lengths, rows, cache)
        call.per_request(batch, (slots, cache.slots - 1, "slots"), (positions, cache.capacity - 1, "positions"),
                         (lengths, rows, "lengths"))
        call.scalars(batch, rows)
        call.run()

    def kv_read_int8(self, cache, slots, positions, lengths, rows):
        """fp16 k, v [B,G,rows,D]: row i < lengths[b] (None: rows) is token positions[b]
        + i of slots[b]; zeros past the length and outside the cache.  slots, positions
        and lengths as in ``kv_append_int8``."""
        torch = self.torch
        call = _Call(self, "ti_amd_kv_read_i8")
        call.cache(cache)
        batch = self._batch_of(slots, positions, lengths)
        _count(rows, "rows")
        self._batch_rows(batch, slots, positions, lengths, rows, cache)
        shape = (batch, cache.kv_heads, rows, cache.head_dim)
        k = call.output(shape, torch.float16)
        v = call.output_like(k)
        call.per_request(batch, (slots, cache.slots - 1, "slots"), (positions, cache.capacity - 1, "positions"),
                         (lengths, rows, "lengths"))
        call.scalars(batch, rows)
        call.run()
        return k, v

    def _batch_of(self, *values):
        for value in values:
            if value is not None and type(value) is not int:
                return len(value)
        return 1

    def _batch_rows(self, batch, slots, positions, lengths, rows, cache):
        """Host positions and lengths must stay inside the cache."""
        if slots is None or positions is None:
            raise ValueError("slots and positions are required")
        if batch > 65535 or rows > 1 << 28:
            raise ValueError("batch must be at most 65535, rows at most 2^28")
        tensor = self.tensor_type
        if isinstance(positions, tensor) or isinstance(lengths, tensor):
            return
        first = _per_request(positions, batch, 0, cache.capacity - 1, "positions")
        count = _per_request(lengths, batch, rows, rows, "lengths")
        if max(map(int.__add__, first, count)) > cache.capacity:
            raise ValueError(f"positions + lengths pass the cache's capacity of {cache.capacity}")

    def attention_int8kv(self, q, cache, slots, kv_lengths, *, q_lengths=None, query_offsets=None, causal=True,
                         max_kv_length=None):
        """q [B,H,Q,D] fp16 over the int8 cache, H a multiple of its key heads (query
        head h reads key head h // (H // G)): request b's keys are tokens 0 ..
        kv_lengths[b] - 1 of slots[b].

        Causal: query i sees keys up to query_offsets[b] + i; None means
        kv_lengths[b] - q_lengths[b], the queries being the request's last tokens
        (append first, then attend).  Rows that see no key and queries past
        q_lengths[b] are 0.  slots, kv_lengths, q_lengths and query_offsets are int32
        [B] tensors or host ints; tensors make a call that a graph can capture.
        max_kv_length: what kv_lengths stay within where the capacity is much larger
        (it plans the launch only)."""
        return self._attend_int8(q, cache, 0, 0, slots, kv_lengths, q_lengths, query_offsets, causal, max_kv_length)

    def attention_shared_prefix(self, q, cache, prefix_slot, prefix_length, slots, kv_lengths, *, q_lengths=None,
                                query_offsets=None, causal=True, max_kv_length=None):
        """``attention_int8kv`` for a batch whose requests share a prefix: in front of its
        own keys every query sees tokens 0 .. prefix_length - 1 (host ints) of
        prefix_slot, which are read once for the whole batch where that is the faster way.  kv_lengths and
        query_offsets count the request's own tokens."""
        if type(cache) is not Int8KVCache:
            raise TypeError("cache: an Int8KVCache (NativeOps.kv_cache_int8) is required")
        _count(prefix_slot, "prefix_slot", 0, cache.slots - 1)
        _count(prefix_length, "prefix_length", 0, cache.capacity)
        return self._attend_int8(q, cache, prefix_slot, prefix_length, slots, kv_lengths, q_lengths, query_offsets,
                                 causal, max_kv_length)

    def _attend_int8(self, q, cache, prefix_slot, prefix_length, slots, kv_lengths, q_lengths, query_offsets, causal,
                     max_kv_length):
        torch = self.torch
        call = _Call(self, "ti_amd_attention_i8kv")
        call.cache(cache)
        call.operand(q, torch.float16, "q", rank=4)
        batch, heads, nq, dim = q.shape
        if dim != cache.head_dim or heads % cache.kv_heads:
            raise ValueError(f"q must be [B, H, Q, {cache.head_dim}] with H a multiple of {cache.kv_heads}, got {list(q.shape)}")
        if batch > 65535 or heads > 65535:
            raise ValueError("batch and heads must each be at most 65535")
        if batch * heads * nq > 1 << 23:
            raise ValueError("at most 2^23 query rows (batch * heads * queries)")
        if type(causal) is not bool:
            raise ValueError("causal must be a bool")
        if slots is None or kv_lengths is None:
            raise ValueError("slots and kv_lengths are required")
        bound = 0 if max_kv_length is None else _count(max_kv_length, "max_kv_length", 0)
        y = call.output_like(q)
        call.per_request(batch, (slots, cache.slots - 1, "slots"), (kv_lengths, cache.capacity, "kv_lengths"),
                         (q_lengths, nq, "q_lengths"), (query_offsets, INT32_MAX - nq, "query_offsets"))
        shape = (batch, heads, nq, bound, prefix_length)
        needed = cache._workspace.get(shape)
        if needed is None:
            if len(cache._workspace) >= 1024:  # (a caller whose lengths are all different)
                cache._workspace.clear()
            needed = cache._workspace[shape] = max(0, self.lib.ti_amd_attention_i8kv_workspace(cache._at, *shape))
        if needed:
            call.output((needed,), torch.uint8)
        else:
            call.args.append(None)
        call.scalars(needed, batch, heads, nq, bound, int(causal), prefix_slot, prefix_length)
        call.run()
        return y

    # -- sampling ----------------------------------------------------------------
    def sample(self, logits, uniforms, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        """One token per row of logits [B,V] (fp16 or fp32) from uniforms fp32 [B] in
        [0, 1): (tokens int32 [B], probs fp32 [B], the tokens' probabilities among the
        kept ones).

        Tokens are ordered by logit, ties by index.  Kept are the first top_k (0: all),
        of these the shortest run from the front with top_p of their probability, of
        these those with at least min_p of the likeliest one's; the token is the first
        whose cumulative probability among them exceeds the row's uniform.  Each of
        temperature, top_p, min_p (fp32) and top_k (int32) is a number for all rows or
        a [B] tensor.  Temperature 0 takes the likeliest token."""
        torch = self.torch
        call = _Call(self, "ti_amd_sample")
        wide = isinstance(logits, self.tensor_type) and logits.dtype == torch.float32
        call.operand(logits, torch.float32 if wide else torch.float16, "logits", rank=2)
        batch, vocab = logits.shape
        if vocab > 1 << 18 or batch > 1 << 20:
            raise ValueError("logits: at most 2^20 rows of 2^18")
        call.scalars(int(wide))
        call.operand(uniforms, torch.float32, "uniforms", shape=(batch,))
        values = []
        for x, dtype, name, high in ((temperature, torch.float32, "temperature", math.inf),
                                     (top_k, torch.int32, "top_k", INT32_MAX), (top_p, torch.float32, "top_p", 1.0),
                                     (min_p, torch.float32, "min_p", 1.0)):
            if isinstance(x, self.tensor_type):
                call.operand(x, dtype, name, shape=(batch,))
                values.append(0)
                continue
            if dtype == torch.int32:
                _count(x, name, 0)
            elif type(x) not in (int, float) or not 0 <= x <= high or x == math.inf:
                raise ValueError(f"{name} must be a number in [0, {'inf)' if high == math.inf else '1]'}")
            call.scalars(None)
            values.append(x)
        call.scalars(*values)
        tokens = call.output((batch,), torch.int32)
        probs = call.output((batch,), torch.float32)
        call.scalars(batch, vocab)
        call.run()
        return tokens, probs

    def logprobs(self, logits, tokens, *, top=0):
        """Log probabilities (natural) under the softmax of each row of logits [B,V] (fp16 or
        fp32): (logprobs of `tokens` int32 [B] or [B,N], in their shape; the rows' entropy
        [B], in nats; top_logprobs [B,top] and top_tokens int32 [B,top], the likeliest tokens
        by logit, ties by index), all fp32 but the last.

        A token outside the vocabulary, or with a logit of -inf or NaN, has the log
        probability -inf and is no alternative: places left over hold 2^31 - 1 and -inf.
        `top` is at most 64; 0 gives two tensors [B,0]."""
        torch = self.torch
        call = _Call(self, "ti_amd_logprobs")
        wide = isinstance(logits, self.tensor_type) and logits.dtype == torch.float32
        call.operand(logits, torch.float32 if wide else torch.float16, "logits", rank=2)
        batch, vocab = logits.shape
        if vocab > 1 << 18 or batch > 1 << 20:
            raise ValueError("logits: at most 2^20 rows of 2^18")
        _count(top, "top", 0, 64)
        call.scalars(int(wide))
        call.operand(tokens, torch.int32, "tokens")
        if tokens.dim() > 2 or tokens.shape[0] != batch or tokens.numel() > batch << 16:
            raise ValueError(f"tokens: shape [{batch}] or [{batch}, N] with N at most 2^16 required, got {list(tokens.shape)}")
        logprobs = call.output(tokens.shape, torch.float32)
        entropy = call.output((batch,), torch.float32)
        if top:
            top_logprobs, top_tokens = call.output((batch, top), torch.float32), call.output((batch, top), torch.int32)
        else:
            top_logprobs, top_tokens = (torch.empty((batch, 0), dtype=d, device=call.device) for d in (torch.float32, torch.int32))
            call.scalars(None, None)
        call.scalars(batch, vocab, tokens.numel() // batch, top)
        call.run()
        return logprobs, entropy, top_logprobs, top_tokens

    # -- rotary positions ----------------------------------------------------------
    def rotary(self, rotated, *, base=10000.0, interleaved=False, scaling=None, factor=1.0, original_length=None, fast=32.0,
               slow=1.0, frequencies=None, amplitude=1.0, device=None):
        """Rotary positions that turn the first `rotated` dims of a row (even), in pairs
        (i, rotated / 2 + i), or (2 i, 2 i + 1) if interleaved, by base^(-2 i / rotated)
        radians a position.

        scaling stretches them for contexts `factor` times as long: "linear" divides every
        frequency by it; "base" multiplies the base by factor^(rotated / (rotated - 2)), so
        that the slowest pair alone is divided; "parts" keeps pairs that turn `fast` times
        or more over original_length, divides those that turn `slow` times or fewer, and
        goes over linearly in the number of turns in between (checkpoints that go over by the
        pairs' numbers give their own frequencies).  frequencies gives all of them instead (radians a
        position, rotated / 2 numbers).  Turned values are multiplied by amplitude."""
        torch = self.torch
        if type(rotated) is not int or rotated < 2 or rotated % 2 or rotated > 65536:
            raise ValueError("rotated must be an even integer in [2, 65536]")
        if type(interleaved) is not bool:
            raise ValueError("interleaved must be a bool")
        _number(base, "base", 0, True)
        _number(factor, "factor", 0, True)
        if abs(_number(amplitude, "amplitude")) > 2.0 ** 128 - 2.0 ** 104:
            raise ValueError("amplitude must be a finite fp32 number")
        if scaling not in (None, "linear", "base", "parts"):
            raise ValueError('scaling must be None, "linear", "base" or "parts"')
        if scaling is None and factor != 1:
            raise ValueError("a factor needs a scaling")
        count = rotated // 2
        if frequencies is not None:
            if scaling is not None or base != 10000.0:
                raise ValueError("frequencies stand in place of a base and a scaling")
            got = [float(_number(f, "frequencies")) for f in frequencies]
            if len(got) != count:
                raise ValueError(f"frequencies must hold {count} numbers, got {len(got)}")
        else:
            if scaling == "parts":
                _count(original_length, "original_length")
                _number(slow, "slow")
                if _number(fast, "fast") <= slow:
                    raise ValueError("fast must be above slow")
            try:
                if scaling == "base" and count > 1:
                    base = base * factor ** (count / (count - 1))
                got = [float(base) ** (-i / count) for i in range(count)]
            except OverflowError:
                got = [math.inf]
            if scaling == "linear":
                got = [f / factor for f in got]
            if scaling == "parts":
                for i, f in enumerate(got):
                    keep = min(max((original_length * f / (2 * math.pi) - slow) / (fast - slow), 0.0), 1.0)
                    got[i] = f * keep + f / factor * (1.0 - keep)
            if not all(map(math.isfinite, got)):
                raise ValueError("base and factor give frequencies beyond every number")
        where = torch.device("cuda" if device is None else device)
        if where.type != "cuda":
            raise TypeError("device: a GPU (torch 'cuda' device) is required")
        return Rotary(torch, got, interleaved, amplitude, where)

    def rotate(self, x, rotary, positions):
        """x fp16 [B,H,Q,D] (its dims contiguous, any other strides) turned by ``rotary``:
        row i of request b at position positions[b] + i.  positions is an int32 [B] tensor,
        host ints (one for all, or B of them), or an int32 [B,Q] tensor with a position for
        every row.  The result is contiguous."""
        call = _Call(self, "ti_amd_rotate")
        self._rotary(rotary)
        batch, heads, rows, dim = call.rows(x, "x", None)
        if rotary.rotated > dim:
            raise ValueError(f"rotary turns {rotary.rotated} dims, x has {dim}")
        if batch > 65535 or heads > 65535 or rows * dim > 1 << 31:
            raise ValueError("x: batch and heads must be at most 65535, rows * dims at most 2^31")
        if positions is None:
            raise ValueError("positions are required")
        y = call.output_like(x)
        each = isinstance(positions, self.tensor_type) and positions.dim() == 2
        if each:
            call.operand(positions, self.torch.int32, "positions", shape=(batch, rows))
        else:
            call.per_request(batch, (positions, INT32_MAX - rows, "positions"))
        call.scalars(int(each))
        call.turn(rotary)
        call.scalars(batch, heads, rows, dim)
        call.run()
        return y

    def _rotary(self, rotary):
        if type(rotary) is not Rotary:
            raise TypeError("rotary: a Rotary (NativeOps.rotary) is required")

    # -- paged KV cache --------------------------------------------------------------
    def kv_cache_paged(self, pages, kv_heads, page_size, head_dim, *, device=None):
        """A zeroed fp16 cache of `pages` pages of `page_size` tokens (a power of two from 32
        to 1024), `kv_heads` key heads of 64 or 128 dims; pages * kv_heads * page_size is at most 2^34."""
        torch = self.torch
        _count(pages, "pages")
        _count(kv_heads, "kv_heads", high=65535)
        if type(page_size) is not int or page_size not in (32, 64, 128, 256, 512, 1024):
            raise ValueError("page_size must be a power of two from 32 to 1024")
        if type(head_dim) is not int or head_dim not in (64, 128):
            raise ValueError("head_dim must be 64 or 128")
        if pages * kv_heads * page_size > 1 << 34:
            raise ValueError("pages * kv_heads * page_size must be at most 2^34")
        where = torch.device("cuda" if device is None else device)
        if where.type != "cuda":
            raise TypeError("device: a GPU (torch 'cuda' device) is required")
        return PagedKVCache(torch, pages, kv_heads, page_size, head_dim, where)

    def kv_append_paged(self, cache, k, v, page_table, positions, *, lengths=None, rotary=None, q=None):
        """Put k, v fp16 [B,G,Q,D] into the cache: row i < lengths[b] (None: Q) becomes token
        positions[b] + i of request b, on the page that page_table (int32 [B,W]) names for it.
        With ``rotary`` (turning a multiple of 16 dims) keys are turned by their positions on
        the way, and so is q fp16 [B,H,Q,D], whose turned rows are returned (zeros past
        lengths[b]); None without q.

        k, v and q may have any strides but the dims', as the slices of one projection do.
        positions and lengths are int32 [B] tensors, or host ints (one for all, or B of them).
        Host values must lie inside the table; rows that device values put outside it, or on a
        page outside the cache, are not written.  Rows of one call must not share a place."""
        call = _Call(self, "ti_amd_kv_append_paged")
        call.cache(cache, PagedKVCache)
        shape = batch, heads, rows, dim = call.rows(k, "k", None)
        if heads != cache.kv_heads or dim != cache.head_dim:
            raise ValueError(f"k must be [B, {cache.kv_heads}, Q, {cache.head_dim}], got {list(k.shape)}")
        call.rows(v, "v", shape)
        if rotary is not None:
            self._rotary(rotary)
            if rotary.rotated % 16 or rotary.rotated > dim:
                raise ValueError(f"rotary must turn a multiple of 16 of the head's {dim} dims, not {rotary.rotated}")
        q_heads, turned = 0, None
        if q is None:
            call.scalars(None, 0, 0, 0, None)
        else:
            if rotary is None:
                raise ValueError("q is only turned: it needs rotary")
            q_shape = q_batch, q_heads, q_rows, q_dim = call.rows(q, "q", None)
            if q_batch != batch or q_rows != rows or q_dim != dim or q_heads > 65535:
                raise ValueError(f"q must be [{batch}, H, {rows}, {dim}] with H at most 65535, got {list(q_shape)}")
            turned = call.output_like(q)
        self._paged_rows(call, cache, page_table, positions, lengths, batch, rows)
        call.turn(rotary)
        call.scalars(batch, q_heads, rows)
        call.run()
        return turned

    def kv_read_paged(self, cache, page_table, positions, lengths, rows):
        """fp16 k, v [B,G,rows,D]: row i < lengths[b] (None: rows) is token positions[b] + i of
        request b; zeros past the length and where no token is.  page_table, positions and
        lengths as in ``kv_append_paged``."""
        torch = self.torch
        call = _Call(self, "ti_amd_kv_read_paged")
        call.cache(cache, PagedKVCache)
        _count(rows, "rows", high=1 << 20)
        if not isinstance(page_table, self.tensor_type):
            raise TypeError("page_table: a GPU (torch 'cuda' device) tensor is required")
        batch = page_table.shape[0] if page_table.dim() else 0
        k = call.output((batch, cache.kv_heads, rows, cache.head_dim), torch.float16)
        v = call.output_like(k)
        self._paged_rows(call, cache, page_table, positions, lengths, batch, rows)
        call.scalars(batch, rows)
        call.run()
        return k, v

    def _paged_rows(self, call, cache, page_table, positions, lengths, batch, rows):
        """The table, positions and lengths; host values must stay inside the table."""
        if positions is None:
            raise ValueError("positions are required")
        if batch > 65535 or rows > 1 << 20:
            raise ValueError("batch must be at most 65535, rows at most 2^20")
        held = min(call.page_table(page_table, batch) * cache.page_size, INT32_MAX)
        tensor = self.tensor_type
        if not isinstance(positions, tensor) and not isinstance(lengths, tensor):
            first = _per_request(positions, batch, 0, held - 1, "positions")
            count = _per_request(lengths, batch, rows, rows, "lengths")
            if max(map(int.__add__, first, count)) > held:
                raise ValueError(f"positions + lengths pass the {held} tokens of the page table")
        call.per_request(batch, (positions, held - 1, "positions"), (lengths, rows, "lengths"))

    def attention_paged(self, q, cache, page_table, kv_lengths, *, q_lengths=None, query_offsets=None, causal=True,
                        max_kv_length=None):
        """q [B,H,Q,D] fp16 over the paged cache, H a multiple of its key heads (query head h
        reads key head h // (H // G)): request b's keys are tokens 0 .. kv_lengths[b] - 1 on
        the pages that page_table (int32 [B,W]) names; those on no page of the cache are not
        seen.

        Causal: query i sees keys up to query_offsets[b] + i; None means
        kv_lengths[b] - q_lengths[b], the queries being the request's last tokens
        (append first, then attend).  Rows that see no key and queries past
        q_lengths[b] are 0.  kv_lengths, q_lengths and query_offsets are int32 [B]
        tensors or host ints; tensors make a call that a graph can capture.
        max_kv_length: what kv_lengths stay within where the table holds much more.  It
        plans the launch only, but without it the plan is for a full table: a token over 300
        keys, 12 heads, takes 8.4 us, with a table for 32768 and no max_kv_length 11.8."""
        call = _Call(self, "ti_amd_attention_paged")
        call.cache(cache, PagedKVCache)
        call.operand(q, self.torch.float16, "q", rank=4)
        batch, heads, nq, dim = q.shape
        if dim != cache.head_dim or heads % cache.kv_heads:
            raise ValueError(f"q must be [B, H, Q, {cache.head_dim}] with H a multiple of {cache.kv_heads}, got {list(q.shape)}")
        if batch > 65535 or heads > 65535:
            raise ValueError("batch and heads must each be at most 65535")
        if batch * heads * nq > 1 << 23:
            raise ValueError("at most 2^23 query rows (batch * heads * queries)")
        if type(causal) is not bool:
            raise ValueError("causal must be a bool")
        if kv_lengths is None:
            raise ValueError("kv_lengths are required")
        bound = 0 if max_kv_length is None else _count(max_kv_length, "max_kv_length", 0)
        y = call.output_like(q)
        width = call.page_table(page_table, batch)
        held = min(width * cache.page_size, INT32_MAX)
        call.per_request(batch, (kv_lengths, held, "kv_lengths"), (q_lengths, nq, "q_lengths"),
                         (query_offsets, INT32_MAX - nq, "query_offsets"))
        shape = (width, batch, heads, nq, bound)
        needed = cache._workspace.get(shape)
        if needed is None:
            if len(cache._workspace) >= 1024:  # (a caller whose lengths are all different)
                cache._workspace.clear()
            needed = cache._workspace[shape] = max(0, self.lib.ti_amd_attention_paged_workspace(cache._at, *shape))
        if needed:
            call.output((needed,), self.torch.uint8)
        else:
            call.args.append(None)
        call.scalars(needed, batch, heads, nq, bound, int(causal))
        call.run()
        return y
