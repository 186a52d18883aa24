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
row of logits.

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
from array import array
from contextlib import nullcontext
from pathlib import Path

from . import BACKEND_LIB, require

INT32_MAX = 2**31 - 1
INT64_MAX = 2**63 - 1

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
    operand that passes every check is accepted by one condition and only a
    refused one goes through the ordered checks that name the reason; outputs
    come from the calling stream's own pool and need no record_stream; the
    device is switched only when it is not current.  ``gemm_int8`` at M = 1,
    768 -> 2304, call after call: 15.6 -> 11.7 us."""

    __slots__ = ("ops", "symbol", "args", "held", "made", "device", "index", "over")

    def __init__(self, ops, symbol):
        self.ops, self.symbol = ops, symbol
        self.args = []
        self.held, self.made = [], []   # the caller's tensors, and this call's own
        self.device = self.index = None
        self.over = None                # the int8 cache it works on

    def operand(self, x, dtype, name, rank=None, shape=None):
        tensor = self.ops.tensor_type
        # (At most INT32_MAX elements: then every extent and the byte count fit.)
        if not ((type(x) is tensor or isinstance(x, tensor)) and x.dtype == dtype
                and x.is_contiguous() and not x.requires_grad and 0 < x.numel() <= INT32_MAX
                and (x.shape == shape if shape is not None else x.dim() == rank if rank is not None else x.dim())
                and x.is_cuda and (self.index is None or x.get_device() == self.index)):
            self._checked(x, dtype, name, rank, shape)
        if self.index is None:
            self.device = x.device
            self.index = x.get_device()
        self.held.append(x)
        self.args.append(x.data_ptr())
        return x

    def _checked(self, x, dtype, name, rank, shape):
        """The operand checks one by one, each with its own exception."""
        torch = self.ops.torch
        if not isinstance(x, torch.Tensor) or x.device.type != "cuda":
            raise TypeError(f"{name}: a GPU (torch 'cuda' device) tensor is required")
        if x.dtype != dtype:
            raise TypeError(f"{name}: dtype {x.dtype} given, {dtype} required")
        if not x.is_contiguous():
            raise TypeError(f"{name}: contiguous row-major storage required")
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

    def output(self, shape, dtype):
        y = self.ops.torch.empty(shape, dtype=dtype, device=self.device)
        self.made.append(y)
        self.args.append(y.data_ptr())
        return y

    def output_like(self, x):
        y = self.ops.torch.empty_like(x)
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

    def cache(self, cache):
        if type(cache) is not Int8KVCache:
            raise TypeError("cache: an Int8KVCache (NativeOps.kv_cache_int8) is required")
        self.device = cache.buffer.device
        self.index = cache.buffer.get_device()
        self.over = cache
        self.args.append(cache._at)

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
        # (The current stream's handle costs a tenth of making its Stream object, which
        # record_stream wants and which stays the same for a handle.)
        handle = ops.stream_handle(index)
        stream = ops.streams.get((index, handle))
        if stream is None:
            stream = ops.streams[index, handle] = cuda.current_stream(index)
        for x in self.held:
            x.record_stream(stream)
        # (The allocator keeps a stream with a block until the block is freed: once does.)
        if self.over is not None and handle not in self.over._streams:
            self.over.buffer.record_stream(stream)
            self.over._streams.add(handle)
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


class NativeOps:
    """Inference-only device ops over the v2 ABI; operands are torch GPU tensors,
    work is queued on the current torch stream of their device."""

    def __init__(self, library_path=None):
        import torch
        self.torch, self.tensor_type = torch, torch.Tensor
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
