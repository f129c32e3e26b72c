"""Host-side matmul interface, mirroring ``adrastea_models/src/kernels.rs``.

``CommonKernels.matmul_f16`` / ``matmul_f16_slow`` keep the reference's names, argument meaning
and error behaviour (kernels.rs:206-213, 753-890): views in, options by value, shape mismatches
raise ``AssertionError`` (the reference ``assert_eq!``-panics), device/launcher errors raise
``AdrasteaError`` (the reference returns ``anyhow::Error``).  ``lower_matmul`` is the pure
lowering of views + options to the 22-scalar argument tuple of the C ABI.

The u8 entry points have no Rust caller in the reference (llama.rs:28-29); their methods here
follow the device kernels' argument lists (matmul_nt_fp16u8.cu:4-12, quantize.cu:3-5,46-48).
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import threading
import warnings
from dataclasses import dataclass, field
from typing import Optional, Tuple

from . import _ffi
from .tensor import TensorLayout, TensorView, _native


class AdrasteaError(RuntimeError):
    def __init__(self, code: int, what: str):
        super().__init__(f"{what}: {_ffi.strerror(code)} (code {code})")
        self.code = code


# ---- option enums (kernels.rs:81-167) ------------------------------------------------------

class MatmulMask:
    NONE = 0
    CAUSAL = 1


@dataclass(frozen=True)
class MatmulLoad:
    op: int = 0          # MatmulLoadOp: Identity = 0, Scale = 1
    scale: float = 1.0

    @staticmethod
    def Identity() -> "MatmulLoad":
        return MatmulLoad(0, 1.0)

    @staticmethod
    def Scale(scale: float) -> "MatmulLoad":
        return MatmulLoad(1, float(scale))

    def lower(self) -> int:
        return self.op


@dataclass(frozen=True)
class MatmulStore:
    op: int = 0          # MatmulStoreOp, kernels.rs:103-112
    beta: float = 0.0
    scale: Optional[float] = None
    bias: Optional[TensorView] = None

    @staticmethod
    def Identity() -> "MatmulStore":
        return MatmulStore(0)

    @staticmethod
    def GeluBias(bias) -> "MatmulStore":
        return MatmulStore(1, bias=bias)

    @staticmethod
    def BetaGeluBias(beta: float, bias) -> "MatmulStore":
        return MatmulStore(2, beta=float(beta), bias=bias)

    @staticmethod
    def BetaBias(beta: float, bias) -> "MatmulStore":
        return MatmulStore(3, beta=float(beta), bias=bias)

    @staticmethod
    def Scale(scale: float) -> "MatmulStore":
        return MatmulStore(4, scale=float(scale))

    @staticmethod
    def Add() -> "MatmulStore":
        return MatmulStore(5)

    @staticmethod
    def QuickGeluBias(bias) -> "MatmulStore":
        return MatmulStore(6, bias=bias)

    def lower(self) -> int:
        return self.op


@dataclass(frozen=True)
class MatmulOptions:
    """Builder with the reference's method names (kernels.rs:143-167)."""
    load_: MatmulLoad = field(default_factory=MatmulLoad.Identity)
    store_: MatmulStore = field(default_factory=MatmulStore.Identity)
    mask_: int = MatmulMask.NONE

    @staticmethod
    def new() -> "MatmulOptions":
        return MatmulOptions()

    def load(self, load: MatmulLoad) -> "MatmulOptions":
        return MatmulOptions(load, self.store_, self.mask_)

    def store(self, store: MatmulStore) -> "MatmulOptions":
        return MatmulOptions(self.load_, store, self.mask_)

    def mask(self, mask: int) -> "MatmulOptions":
        return MatmulOptions(self.load_, self.store_, mask)


# ---- lowering (kernels.rs:821-890) -----------------------------------------------------------

@dataclass(frozen=True)
class LoweredMatmul:
    batches: int
    m: int
    k: int
    n: int
    stride_o: Tuple[int, int, int]   # (x, y, z)
    stride_l: Tuple[int, int, int]
    stride_r: Tuple[int, int, int]
    beta: float
    scale: float
    store: int
    load: int
    mask: int

    def scalars(self):
        return (self.batches, self.m, self.k, self.n, *self.stride_o, *self.stride_l,
                *self.stride_r)


def _lower(output: TensorLayout, left: TensorLayout, right: TensorLayout, options: MatmulOptions):
    """The 13 shape and stride scalars of the C ABI, and (beta, scale, store, load, mask)."""
    od, ld, rd = output.dims, left.dims, right.dims
    m, k, n = ld[-2], ld[-1], rd[-1]
    assert k == rd[-2], "K mismatch"                           # kernels.rs:825
    assert od[-2] == m, "M mismatch"                           # kernels.rs:826
    assert od[-1] == n, "N mismatch"                           # kernels.rs:827
    load, store = options.load_, options.store_
    scale = load.scale if load.op == 1 else 1.0
    if store.op == 4:
        scale *= store.scale                                   # one float for both (:837-843)
    beta = store.beta if store.op in (2, 3) else 0.0
    os, ls, rs = output.strides, left.strides, right.strides
    # batch stride 0 for rank-2 operands: they are broadcast over the batches (kernels.rs:868-880)
    return ((od[-3] if len(od) > 2 else 1, m, k, n,
             os[-1], os[-2], os[-3] if len(od) > 2 else 0,
             ls[-1], ls[-2], ls[-3] if len(ld) > 2 else 0,
             rs[-1], rs[-2], rs[-3] if len(rd) > 2 else 0),
            (beta, scale, store.lower(), load.lower(), options.mask_))


def lower_matmul(output: TensorLayout, left: TensorLayout, right: TensorLayout,
                 options: MatmulOptions) -> LoweredMatmul:
    s, tail = _lower(output, left, right, options)
    return LoweredMatmul(*s[:4], s[4:7], s[7:10], s[10:], *tail)


# ---- several sequences at once ---------------------------------------------------------------

class RotaryLayout:
    HALVES = 0   # value i is paired with value i + dims / 2
    PAIRS = 1    # value 2 i with value 2 i + 1


@dataclass(frozen=True)
class RotaryScaling:
    """How the frequencies base^(-2 i / dims) are changed for contexts longer than a model was trained on."""
    kind: str = "identity"
    parameters: Tuple[float, ...] = ()

    @staticmethod
    def Identity() -> "RotaryScaling":
        return RotaryScaling()

    @staticmethod
    def Linear(factor: float) -> "RotaryScaling":
        """Positions divided by `factor`."""
        return RotaryScaling("linear", (float(factor),))

    @staticmethod
    def Base(factor: float) -> "RotaryScaling":
        """The base grown so that the slowest pair turns `factor` times slower and the fastest as before."""
        return RotaryScaling("base", (float(factor),))

    @staticmethod
    def Wavelength(factor: float, low: float, high: float, original: int) -> "RotaryScaling":
        """Pairs that turn fewer than `low` times within `original` positions are slowed by `factor`, those that turn
        more than `high` times are not, and those between are blended by their number of turns."""
        return RotaryScaling("wavelength", (float(factor), float(low), float(high), float(original)))

    @staticmethod
    def Yarn(factor: float, original: int, fast: float = 32.0, slow: float = 1.0,
             magnitude: Optional[float] = None) -> "RotaryScaling":
        """A ramp over the pairs' indices, from the pair that turns `fast` times within `original` positions (kept) to
        the one that turns `slow` times (slowed by `factor`), and the rotated values multiplied by `magnitude`
        (default 0.1 ln(factor) + 1)."""
        if magnitude is None:
            magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
        return RotaryScaling("yarn", (float(factor), float(original), float(fast), float(slow), float(magnitude)))


def rotary_frequencies(dims: int, base: float = 10000.0, scaling: RotaryScaling = RotaryScaling()):
    """(radians a position for each of the dims / 2 pairs, magnitude), in Python's 64-bit floats."""
    if dims < 0 or dims % 2 or not base > 0.0:
        raise ValueError("rotary positions need an even number of values and a positive base")
    p = scaling.parameters
    if p and not p[0] > 0.0:
        raise ValueError("the factor of a scaling is positive")
    if scaling.kind == "base" and dims > 2:
        base *= p[0] ** (dims / (dims - 2))
    f = [base ** (-2.0 * i / dims) for i in range(dims // 2)]
    if scaling.kind == "linear":
        return [x / p[0] for x in f], 1.0
    if scaling.kind == "wavelength":
        factor, low, high, original = p
        if not high > low:
            raise ValueError("wavelength scaling needs high > low")
        keep = [min(max((original * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
        return [x * (k + (1.0 - k) / factor) for x, k in zip(f, keep)], 1.0
    if scaling.kind == "yarn":
        factor, original, fast, slow, magnitude = p

        def index(turns):  # of the pair that turns so many times within the original context
            return dims * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), dims - 1)
        slowed = [min(max((i - low) / max(high - low, 0.001), 0.0), 1.0) for i in range(dims // 2)]
        return [x * (1.0 - s + s / factor) for x, s in zip(f, slowed)], magnitude
    if scaling.kind not in ("identity", "base"):
        raise ValueError(f"unknown rotary scaling {scaling.kind!r}")
    return f, 1.0


@dataclass(frozen=True)
class Rotary:
    """Rotary positions of a model: its frequencies in turns a position, on the device, made once."""
    turns: object        # float64 tensor [dims / 2]
    layout: int = RotaryLayout.HALVES
    magnitude: float = 1.0

    def __post_init__(self):
        import torch
        assert self.turns.dtype == torch.float64 and self.turns.dim() == 1 and self.turns.is_contiguous(), \
            "turns: a contiguous float64 tensor of rank 1"

    @staticmethod
    def new(dims: int, base: float = 10000.0, layout: int = RotaryLayout.HALVES,
            scaling: RotaryScaling = RotaryScaling()) -> "Rotary":
        import torch
        frequencies, magnitude = rotary_frequencies(dims, base, scaling)
        turns = torch.tensor([f / (2 * math.pi) for f in frequencies], dtype=torch.float64).cuda()
        return Rotary(turns, layout, magnitude)

    @property
    def _desc(self) -> _ffi.RotaryDesc:
        _here(self.turns)
        _int32("turns", 2 * self.turns.numel())
        return _ffi.RotaryDesc(self.turns.data_ptr(), 2 * self.turns.numel(), self.layout, self.magnitude)


_NO_ROTARY = _ffi.RotaryDesc(None, 0, 0, 1.0)


@dataclass(frozen=True)
class PagedCache:
    """Keys and values of many sequences in pages: two [pages, kv_heads, page_size, d] views of the pools that
    the program owns (a pool kept as [pages, page_size, kv_heads, d] is handed over as its permuted view)."""
    key: TensorView
    value: TensorView

    def __post_init__(self):
        k, v = self.key.layout, self.value.layout
        assert len(k.dims) == 4 and k.dims == v.dims, "key and value pages are [pages, kv_heads, page_size, d] views"
        _halves("key pages", self.key)
        _halves("value pages", self.value)

    @property
    def _desc(self) -> _ffi.PagedCacheDesc:
        k, v = self.key.layout, self.value.layout
        _here(self.key.storage, self.value.storage)
        p, h, s, d = k.dims
        _int32("sizes of the pages", p, h, s, d)
        return _ffi.PagedCacheDesc(self.key.data_ptr(), self.value.data_ptr(), p, h, s, d,
                                   *(t.strides[i] for t in (k, v) for i in (3, 2, 1, 0)))


def _here(*storages) -> None:
    """Device memory of the current device: what a launch there may be given."""
    import torch
    device = torch.cuda.current_device()
    for s in storages:
        at = getattr(s, "get_device", None)
        assert at is None or at() == device, f"memory of device {at()} in a call on device {device} (-1: the host)"


def _int32(what: str, *values: int) -> None:
    """The C interface has 32 bits for them, and ctypes drops the others without a word."""
    for v in values:
        if not -2 ** 31 <= v < 2 ** 31:
            raise ValueError(f"{what}: {v} does not fit 32 bits")


def _halves(what: str, view) -> None:
    """Values of fp16, or their bits in 16-bit integers: the kernels would read and write any other type as if it were."""
    import torch
    dtype = getattr(view.storage, "dtype", None)
    if dtype not in (torch.float16, torch.int16, torch.uint16) and (dtype is not None or view.storage.element_size() != 2):
        raise TypeError(f"{what}: values of {dtype}, not of fp16")


def _hint(v: int) -> int:
    """(Hints choose kernels and nothing else: what is too large for 32 bits says the same as their largest number.)"""
    return min(max(v, -2 ** 31), 2 ** 31 - 1)


def _index(t, rank, what):
    import torch
    assert t.dtype == torch.int32 and t.dim() == rank and (t.numel() == 0 or t.stride(-1) == 1), \
        f"{what}: an int32 tensor of rank {rank}, contiguous in its last dimension"
    return t


@dataclass(frozen=True)
class PagedBatch:
    """The sequences of one step over a paged cache: rows row_offsets[s] .. row_offsets[s + 1] - 1 belong to sequence s,
    which has lengths[s] keys in the cache with those of this step, on the pages of table[s].  int32 tensors on the
    device, which a program may refill from step to step (and between replays of a captured graph); longest_rows and
    longest are what the host knows of the most rows and keys of a sequence (0: nothing), and only choose kernels."""
    row_offsets: object  # [sequences + 1]
    lengths: object      # [sequences]
    table: object        # [sequences, pages of the longest]
    longest_rows: int = 0
    longest: int = 0

    def __post_init__(self):
        n = _index(self.lengths, 1, "lengths").shape[0]
        assert _index(self.row_offsets, 1, "row_offsets").shape[0] == n + 1, "row_offsets has one entry more than lengths"
        assert _index(self.table, 2, "table").shape[0] == n, "table has a row for each sequence"

    @property
    def _desc(self) -> _ffi.PagedBatchDesc:
        n = self.lengths.shape[0]
        _here(self.row_offsets, self.lengths, self.table)
        pitch = self.table.stride(0) if n > 1 else self.table.shape[1]
        _int32("sequences and table", n, self.table.shape[1], pitch)
        return _ffi.PagedBatchDesc(self.row_offsets.data_ptr(), self.lengths.data_ptr(), self.table.data_ptr(), n,
                                   self.table.shape[1], pitch, _hint(self.longest_rows), _hint(self.longest))


@dataclass(frozen=True)
class PackedBatch:
    """Sequences whose rows, and whose keys, lie one behind the other (whole prompts: the same offsets twice)."""
    row_offsets: object  # [sequences + 1]
    key_offsets: object  # [sequences + 1]
    longest_rows: int = 0
    longest: int = 0

    def __post_init__(self):
        n = _index(self.row_offsets, 1, "row_offsets").shape[0]
        assert n >= 1 and _index(self.key_offsets, 1, "key_offsets").shape[0] == n, "offsets of the same sequences"

    @property
    def _desc(self) -> _ffi.PackedBatchDesc:
        n = self.row_offsets.shape[0]
        _here(self.row_offsets, self.key_offsets)
        _int32("sequences", n)
        return _ffi.PackedBatchDesc(self.row_offsets.data_ptr(), self.key_offsets.data_ptr(), n - 1, _hint(self.longest_rows),
                                    _hint(self.longest))


def _rows_view(view: TensorView, what: str):
    """(heads, rows, d), (x, y, z) strides of a [heads, rows, d] view; rank 2: one head."""
    dims, strides = view.layout.dims, view.layout.strides
    assert len(dims) in (2, 3), f"{what}: a [heads, rows, d] view"
    _here(view.storage)
    _halves(what, view)
    # (of a dimension of one the stride is never used, and may be anything)
    strides = tuple(0 if n <= 1 and not -2 ** 31 <= s < 2 ** 31 else s for n, s in zip(dims, strides))
    _int32(what, *dims, *strides)
    if len(dims) == 2:
        return (1, *dims), (strides[1], strides[0], 0)
    return dims, strides[::-1]


# ---- the kernel interface ----------------------------------------------------------------------

class CommonKernels:
    """The matmul subset of the reference trait (kernels.rs:169-229)."""

    def matmul_f16(self, output: TensorView, left: TensorView, right: TensorView,
                   options: MatmulOptions) -> None:
        raise NotImplementedError

    def matmul_f16_slow(self, output: TensorView, left: TensorView, right: TensorView,
                        options: MatmulOptions) -> None:
        raise NotImplementedError

    def softmax_rows_inplace(self, output: TensorView, temperature: float) -> None:
        raise NotImplementedError


def _current_stream() -> int:
    import torch
    # (the handle torch.cuda.current_stream().cuda_stream gives, without the Stream object made to
    # ask it: 2.7 -> 0.4 us a call)
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


_NATIVE_CALLS = ("adr_matmul_f16", "adr_attention_f16", "adr_softmax_rows", "adr_matmul_nt_fp16u8",
                 "adr_quantize_absmax_u8", "adr_dequantize_absmax_u8", "adr_error_stats_f16", "adr_error_stats_f32")


@functools.lru_cache(maxsize=None)
def _native_binding() -> tuple:
    """The library's functions and torch's for the native host path (ctypes takes 20 us to find the addresses)."""
    import torch
    lib = _ffi.lib()
    return (lib.adr_abi_version(), *(C.cast(getattr(lib, name), C.c_void_p).value for name in _NATIVE_CALLS),
            torch.cuda.current_device, torch._C._cuda_getCurrentRawStream)


_NATIVE_SEQUENCE_CALLS = ("adr_rotary_f16", "adr_append_f16", "adr_attention_paged_f16", "adr_attention_packed_f16")


@functools.lru_cache(maxsize=None)
def _native_sequence_binding() -> tuple:
    import torch
    lib = _ffi.lib()
    return (*(C.cast(getattr(lib, name), C.c_void_p).value for name in _NATIVE_SEQUENCE_CALLS), torch.int32)


def _bind_native() -> None:
    _native.bind(*_native_binding())
    _native.bind_sequences(*_native_sequence_binding())


class GpuKernels(CommonKernels):
    """Launches through the C ABI on torch's current HIP stream.

    Where host/native.cpp is built, the calls below are lowered by it; what it does not take (it
    returns None) goes the way written out here, which is also the definition of what it does.
    Without it every call goes that way, and the constructor warns.

    `workspace_bytes` > 0 gives the instance a scratch buffer of that size, owned like any other
    tensor of the host (in the reference: one more GpuBuffer held by GpuKernels); matmul_f16 then
    goes through adr_matmul_f16_ws, which may split K over workgroups for products with few
    output tiles and a long K, and attention_f16 through adr_attention_f16_ws, which may share keys
    over workgroups for few query rows.  The buffer carries nothing between calls; one instance must
    not be used from streams that run concurrently.  Without it (the default) the library takes such
    a buffer from its own per-stream cache (set_held_workspace_limit)."""

    def __init__(self, workspace_bytes: int = 0):
        self._lib = _ffi.lib()
        import torch
        if not torch.cuda.is_available():
            raise RuntimeError("adrastea_amd.GpuKernels needs a GPU; there is no CPU fallback")
        self._workspace = (torch.empty(workspace_bytes, dtype=torch.uint8, device="cuda")
                           if workspace_bytes > 0 else None)
        if _native is not None:
            _bind_native()
        else:
            warnings.warn("adrastea_amd._native is not built for this interpreter: the calls take 2-10 us more of the host "
                          "each (`python -m adrastea_amd.build`)", RuntimeWarning, stacklevel=2)

    @staticmethod
    def _lowered(name, *args) -> bool:
        """The call as native code; False: it has to go the general way."""
        if _native is None:
            return False
        rc = getattr(_native, name)(*args)
        if rc:
            raise AdrasteaError(rc, name)
        return rc == 0

    def _matmul(self, fn, what, output, left, right, options):
        scalars, tail = _lower(output.layout, left.layout, right.layout, options)
        bias = options.store_.bias
        rc = fn(_current_stream(), output.data_ptr(), left.data_ptr(), right.data_ptr(), *scalars,
                bias.data_ptr() if bias is not None else None, *tail)
        if rc != 0:
            raise AdrasteaError(rc, what)

    def matmul_f16(self, output, left, right, options=MatmulOptions()):
        if self._workspace is None:
            if self._lowered("matmul_f16", output, left, right, options):
                return
            return self._matmul(self._lib.adr_matmul_f16, "matmul_f16", output, left, right, options)
        ws = self._workspace

        def with_workspace(*args):
            return self._lib.adr_matmul_f16_ws(*args, ws.data_ptr(), ws.numel())
        self._matmul(with_workspace, "matmul_f16", output, left, right, options)

    def matmul_f16_slow(self, output, left, right, options=MatmulOptions()):
        self._matmul(self._lib.adr_matmul_f16_slow, "matmul_f16_slow", output, left, right,
                     options)

    def softmax_rows_inplace(self, output, temperature: float = 1.0):
        """kernels.rs:892-915: rows = size(-2), heads = size(-3) (1 for rank 2), width size(-1);
        like the reference's kernel, the tensor is taken to be contiguous."""
        if self._lowered("softmax_rows_inplace", output, temperature):
            return
        lay = output.layout
        assert lay == TensorLayout.row_major(list(lay.dims)), "softmax_rows needs a contiguous view"
        heads = lay.size(-3) if len(lay.dims) > 2 else 1
        rc = self._lib.adr_softmax_rows(_current_stream(), output.data_ptr(), output.data_ptr(),
                                        heads, lay.size(-2), lay.size(-1), float(temperature))
        if rc != 0:
            raise AdrasteaError(rc, "softmax_rows_inplace")

    def attention_f16(self, output, query, key, value, scale: float, temperature: float = 1.0,
                      mask: int = MatmulMask.NONE):
        """The three calls of llama.rs:541-554 (QK^T with Scale and the mask, softmax_rows_inplace,
        P.V) as one call that keeps the scores out of memory.  `query`/`output` are
        [heads, m, d] views, `key`/`value` [heads, n, d] views (rank 2 = one head).  Raises
        AdrasteaError with code ADR_EUNSUPPORTED_LAYOUT for head dimensions or strides the fused
        kernel does not cover; the three-call sequence remains available for those."""
        if self._workspace is None and self._lowered("attention_f16", output, query, key, value, scale, temperature, mask):
            return
        lo, lq, lk, lv = output.layout, query.layout, key.layout, value.layout
        do, dq, dk, dv = lo.dims, lq.dims, lk.dims, lv.dims
        so, sq, sk, sv = lo.strides, lq.strides, lk.strides, lv.strides
        rank = len(dq)
        assert rank in (2, 3) and len(do) == rank and len(dk) == rank and len(dv) == rank
        m, d, n = dq[-2], dq[-1], dk[-2]
        assert dk[-1] == d and dv[-1] == d and dv[-2] == n
        assert do[-2] == m and do[-1] == d
        heads, zo, zq, zk, zv = 1, 0, 0, 0, 0
        if rank == 3:
            heads, zo, zq, zk, zv = dq[0], so[0], sq[0], sk[0], sv[0]
            assert do[0] == heads and dk[0] == heads and dv[0] == heads
        args = (_current_stream(), output.data_ptr(), query.data_ptr(), key.data_ptr(), value.data_ptr(), heads, m, n, d,
                so[-1], so[-2], zo, sq[-1], sq[-2], zq, sk[-1], sk[-2], zk, sv[-1], sv[-2], zv,
                float(scale), float(temperature), int(mask))
        ws = self._workspace
        rc = (self._lib.adr_attention_f16(*args) if ws is None else
              self._lib.adr_attention_f16_ws(*args, ws.data_ptr(), ws.numel()))
        if rc != 0:
            raise AdrasteaError(rc, "attention_f16")

    # -- several sequences at once --
    def rotary_f16(self, output, input, positions, rotary: Rotary):
        """The rows of `input`, a [heads, rows, d] view, turned by positions[row] into `output` (which may be the same
        view).  positions: int32 [rows]."""
        if self._lowered("rotary_f16", output, input, positions, rotary):
            return
        dims, si = _rows_view(input, "input")
        dims_out, so = _rows_view(output, "output")
        assert dims_out == dims, "output and input have one shape"
        assert _index(positions, 1, "positions").shape[0] == dims[1], "a position for each row"
        _here(positions)
        rc = self._lib.adr_rotary_f16(_current_stream(), output.data_ptr(), input.data_ptr(), positions.data_ptr(),
                                      rotary._desc, *dims, *so, *si)
        if rc != 0:
            raise AdrasteaError(rc, "rotary_f16")

    def append_f16(self, cache: PagedCache, batch: PagedBatch, key, value, rotary: Optional[Rotary] = None,
                   query_out=None, query=None, positions=None):
        """The step's keys, turned, and values ([kv_heads, rows, d] views) into their pages, and its queries ([heads,
        rows, d]) turned into `query_out`, which may be the same view.  Row j of the r of sequence s goes to
        place lengths[s] - r + j and is turned by it, or by positions[row] (int32 [rows])."""
        if self._lowered("append_f16", cache, batch, key, value, rotary, query_out, query, positions):
            return
        c, b = cache._desc, batch._desc
        dims, sk = _rows_view(key, "key")
        dims_v, sv = _rows_view(value, "value")
        assert dims_v == dims and dims[0] == c.kv_heads and dims[2] == c.d, "key and value are [kv_heads, rows, d] views"
        heads, sq, so = 0, (0, 0, 0), (0, 0, 0)
        assert (query is None) == (query_out is None), "query and query_out go together"
        if query is not None:
            dims_q, sq = _rows_view(query, "query")
            dims_o, so = _rows_view(query_out, "query_out")
            heads = dims_q[0]
            assert dims_o == dims_q and dims_q[1:] == dims[1:], "query and query_out are [heads, rows, d] views"
        if positions is not None:
            assert _index(positions, 1, "positions").shape[0] == dims[1], "a position for each row"
            _here(positions)
        rc = self._lib.adr_append_f16(
            _current_stream(), c, b, key.data_ptr(), value.data_ptr(), query_out.data_ptr() if heads else None,
            query.data_ptr() if heads else None, positions.data_ptr() if positions is not None else None,
            rotary._desc if rotary is not None else _NO_ROTARY, heads, dims[1], *sk, *sv, *so, *sq)
        if rc != 0:
            raise AdrasteaError(rc, "append_f16")

    def attention_paged_f16(self, output, query, cache: PagedCache, batch: PagedBatch, scale: float,
                            temperature: float = 1.0, mask: int = MatmulMask.CAUSAL):
        """Attention of the step's rows ([heads, rows, d] views) over the cache: query head h reads key head
        h / (heads / kv_heads), and under the mask the last row of a sequence sees all its keys."""
        if self._workspace is None and self._lowered("attention_paged_f16", output, query, cache, batch, scale, temperature, mask):
            return
        c, b = cache._desc, batch._desc
        dims, sq = _rows_view(query, "query")
        dims_o, so = _rows_view(output, "output")
        assert dims_o == dims and dims[2] == c.d, "output and query are [heads, rows, d] views"
        args = (_current_stream(), output.data_ptr(), query.data_ptr(), c, b, dims[0], dims[1], *so, *sq, float(scale),
                float(temperature), int(mask))
        ws = self._workspace
        rc = (self._lib.adr_attention_paged_f16(*args) if ws is None else
              self._lib.adr_attention_paged_f16_ws(*args, ws.data_ptr(), ws.numel()))
        if rc != 0:
            raise AdrasteaError(rc, "attention_paged_f16")

    def attention_packed_f16(self, output, query, key, value, batch: PackedBatch, scale: float,
                             temperature: float = 1.0, mask: int = MatmulMask.CAUSAL):
        """Attention of packed rows ([heads, rows, d] views) over packed keys and values ([kv_heads, keys, d])."""
        if self._workspace is None and self._lowered("attention_packed_f16", output, query, key, value, batch, scale,
                                                     temperature, mask):
            return
        dims, sq = _rows_view(query, "query")
        dims_o, so = _rows_view(output, "output")
        dims_k, sk = _rows_view(key, "key")
        dims_v, sv = _rows_view(value, "value")
        assert dims_o == dims, "output and query are [heads, rows, d] views"
        assert dims_v == dims_k and dims_k[2] == dims[2], "key and value are [kv_heads, keys, d] views"
        args = (_current_stream(), output.data_ptr(), query.data_ptr(), key.data_ptr(), value.data_ptr(), batch._desc,
                dims[0], dims_k[0], dims[1], dims_k[1], dims[2], *so, *sq, *sk, *sv, float(scale), float(temperature),
                int(mask))
        ws = self._workspace
        rc = (self._lib.adr_attention_packed_f16(*args) if ws is None else
              self._lib.adr_attention_packed_f16_ws(*args, ws.data_ptr(), ws.numel()))
        if rc != 0:
            raise AdrasteaError(rc, "attention_packed_f16")

    def _error_stats(self, fn, what, output, lhs, rhs):
        if _native is not None:
            rc = _native.error_stats(output, lhs, rhs, int(what == "error_stats_f32"))
            if rc:
                raise AdrasteaError(rc, what)
            if rc == 0:
                return
        # kernels.rs:717-751: both operands flattened with shape_cast(&[-1]); equal lengths
        lhs, rhs = lhs.shape_cast([-1]), rhs.shape_cast([-1])
        assert lhs.size(-1) == rhs.size(-1)
        rc = fn(_current_stream(), descriptor(output), descriptor(lhs), descriptor(rhs))
        if rc != 0:
            raise AdrasteaError(rc, what)

    def error_stats_f16(self, output, lhs, rhs):
        self._error_stats(self._lib.adr_error_stats_f16, "error_stats_f16", output, lhs, rhs)

    def error_stats_f32(self, output, lhs, rhs):
        self._error_stats(self._lib.adr_error_stats_f32, "error_stats_f32", output, lhs, rhs)

    # -- contiguous NT forms (device signatures only in the reference) --
    def matmul_nt_f16(self, output, lhs, rhs, beta: float = 0.0):
        m, p = lhs.shape
        n = rhs.shape[0]
        assert rhs.shape[1] == p and tuple(output.shape) == (m, n)
        assert output.is_contiguous() and lhs.is_contiguous() and rhs.is_contiguous()
        rc = self._lib.adr_matmul_nt_f16(_current_stream(), output.data_ptr(), lhs.data_ptr(),
                                         rhs.data_ptr(), m, p, n, beta)
        if rc != 0:
            raise AdrasteaError(rc, "matmul_nt_f16")

    def matmul_nt_fp16u8(self, output, lhs, rhs_q, scales, block_size: int, beta: float = 0.0):
        if self._workspace is None and self._lowered("matmul_nt_fp16u8", output, lhs, rhs_q, scales, block_size, beta):
            return
        m, p = lhs.shape
        n = rhs_q.shape[0]
        assert rhs_q.shape[1] == p and tuple(output.shape) == (m, n)
        assert tuple(scales.shape) == (n, p // block_size)
        assert all(t.is_contiguous() for t in (output, lhs, rhs_q, scales))
        if self._workspace is None:
            rc = self._lib.adr_matmul_nt_fp16u8(_current_stream(), output.data_ptr(), lhs.data_ptr(),
                                                rhs_q.data_ptr(), scales.data_ptr(), m, p, n,
                                                block_size, beta)
        else:
            # with a workspace of n * p * 2 bytes or more, products of 768 rows and more dequantise
            # the matrix once and run the fp16 kernels (same bits)
            rc = self._lib.adr_matmul_nt_fp16u8_ws(_current_stream(), output.data_ptr(), lhs.data_ptr(),
                                                   rhs_q.data_ptr(), scales.data_ptr(), m, p, n,
                                                   block_size, beta, self._workspace.data_ptr(),
                                                   self._workspace.numel())
        if rc != 0:
            raise AdrasteaError(rc, "matmul_nt_fp16u8")

    def dequantize_absmax_uint8(self, output, scales, q):
        if self._lowered("dequantize_absmax_uint8", output, scales, q):
            return
        rows, cols = q.shape
        block_size = cols // scales.shape[1]
        rc = self._lib.adr_dequantize_absmax_u8(_current_stream(), output.data_ptr(),
                                                q.data_ptr(), scales.data_ptr(), rows, cols,
                                                block_size)
        if rc != 0:
            raise AdrasteaError(rc, "dequantize_absmax_uint8")

    def quantize_absmax_uint8(self, q, scales, x):
        if self._lowered("quantize_absmax_uint8", q, scales, x):
            return
        rows, cols = x.shape
        block_size = cols // scales.shape[1]
        rc = self._lib.adr_quantize_absmax_u8(_current_stream(), q.data_ptr(), scales.data_ptr(),
                                              x.data_ptr(), rows, cols, block_size)
        if rc != 0:
            raise AdrasteaError(rc, "quantize_absmax_uint8")

    def embed_uint8(self, output, ids, table, scales, block_size: int):
        """embed_uint8.cu:3-19: output[t] = dequantised row ids[t] of the u8 table; `ids` is an
        int16 tensor, as the reference's kernel takes them."""
        import torch
        assert ids.dtype == torch.int16 and table.dtype == torch.uint8
        n_ids, n_dim = ids.numel(), table.shape[1]
        assert tuple(output.shape) == (n_ids, n_dim)
        assert tuple(scales.shape) == (table.shape[0], n_dim // block_size)
        assert all(t.is_contiguous() for t in (output, ids, table, scales))
        rc = self._lib.adr_embed_uint8(_current_stream(), n_dim, n_ids, ids.data_ptr(),
                                       output.data_ptr(), table.data_ptr(), scales.data_ptr(),
                                       block_size)
        if rc != 0:
            raise AdrasteaError(rc, "embed_uint8")


def descriptor(view: TensorView) -> _ffi.TensorDesc:
    """TensorGpuDescriptor::from (kernels.rs:38-55): dims and strides reversed, innermost first."""
    d = _ffi.TensorDesc()
    d.ptr = view.data_ptr()
    d.dims = len(view.layout.dims)
    for i, (dim, stride) in enumerate(zip(reversed(view.layout.dims),
                                          reversed(view.layout.strides))):
        d.shape[i] = dim
        d.strides[i] = stride
    return d


def plan_matmul(output: TensorLayout, left: TensorLayout, right: TensorLayout,
                options: MatmulOptions = MatmulOptions(), workspace_bytes: int = 0) -> str:
    """Name of the kernel adr_matmul_f16 (or, with a workspace, adr_matmul_f16_ws) selects for
    these layouts (no device needed)."""
    low = lower_matmul(output, left, right, options)
    buf = C.create_string_buffer(96)
    rc = _ffi.lib().adr_matmul_f16_ws_plan(buf, 96, *low.scalars(), low.store, low.load, low.mask,
                                           int(workspace_bytes))
    if rc != 0:
        raise AdrasteaError(rc, "matmul_f16_plan")
    return buf.value.decode()


def matmul_workspace_bytes(output: TensorLayout, left: TensorLayout, right: TensorLayout,
                           options: MatmulOptions = MatmulOptions()) -> int:
    """Scratch bytes adr_matmul_f16_ws would use for these layouts (0: it would not split K)."""
    low = lower_matmul(output, left, right, options)
    n = _ffi.lib().adr_matmul_f16_workspace_bytes(*low.scalars(), low.store, low.load, low.mask)
    if n < 0:
        raise AdrasteaError(int(n), "matmul_f16_workspace_bytes")
    return int(n)


def attention_workspace_bytes(output: TensorLayout, query: TensorLayout, key: TensorLayout, value: TensorLayout,
                              mask: int = MatmulMask.NONE) -> int:
    """Scratch bytes adr_attention_f16_ws would use for these layouts (0: it would share no keys)."""
    layouts, dims = (output, query, key, value), query.dims
    rank = len(dims)
    strides = [s for l in layouts for s in (l.strides[-1], l.strides[-2], l.strides[0] if rank == 3 else 0)]
    n = _ffi.lib().adr_attention_f16_workspace_bytes(dims[0] if rank == 3 else 1, dims[-2], key.dims[-2], dims[-1],
                                                     *strides, int(mask))
    if n < 0:
        raise AdrasteaError(int(n), "attention_f16_workspace_bytes")
    return int(n)


def attention_paged_workspace_bytes(cache: PagedCache, batch: PagedBatch, heads: int, rows: int) -> int:
    """Scratch bytes adr_attention_paged_f16_ws would use for `rows` packed rows of `heads` query heads (0: it would share no
    keys)."""
    _int32("heads and rows", heads, rows)
    n = _ffi.lib().adr_attention_paged_f16_workspace_bytes(cache._desc, batch._desc, heads, rows)
    if n < 0:
        raise AdrasteaError(int(n), "attention_paged_f16_workspace_bytes")
    return int(n)


def attention_packed_workspace_bytes(batch: PackedBatch, heads: int, kv_heads: int, rows: int, keys: int, d: int) -> int:
    """Scratch bytes adr_attention_packed_f16_ws would use for these sizes (0: it would share no keys)."""
    _int32("heads, rows and keys", heads, kv_heads, rows, keys, d)
    n = _ffi.lib().adr_attention_packed_f16_workspace_bytes(batch._desc, heads, kv_heads, rows, keys, d)
    if n < 0:
        raise AdrasteaError(int(n), "attention_packed_f16_workspace_bytes")
    return int(n)


def set_held_workspace_limit(nbytes: int) -> None:
    """Bytes per buffer of the workspace pool that adr_matmul_f16, adr_matmul_nt_f16, adr_attention_f16, adr_attention_paged_f16 and
    adr_attention_packed_f16 (and, on request, adr_matmul_nt_fp16u8) draw from, one buffer per (device, stream); 0 switches it off."""
    rc = _ffi.lib().adr_set_held_workspace_limit(int(nbytes))
    if rc != 0:
        raise AdrasteaError(int(rc), "set_held_workspace_limit")


def held_workspace_limit() -> int:
    return int(_ffi.lib().adr_held_workspace_limit())


def held_workspace_bytes() -> int:
    """Bytes the pool holds now."""
    return int(_ffi.lib().adr_held_workspace_bytes())


def held_workspace_declined() -> int:
    """Calls so far that wanted a buffer of the pool and ran without one."""
    return int(_ffi.lib().adr_held_workspace_declined())


def release_held_workspace(stream=None) -> None:
    """Frees the pool's buffers of `stream` (a raw stream handle; default: torch's current stream)
    and those no stream owns any more, after waiting for the last launches that used them.  Call it
    before destroying a stream, not while it is being captured.  `stream="all"`: every buffer on
    every device."""
    L = _ffi.lib()
    rc = (L.adr_release_held_workspace_all() if stream == "all" else
          L.adr_release_held_workspace(_current_stream() if stream is None else stream))
    if rc != 0:
        raise AdrasteaError(int(rc), "release_held_workspace")


def set_u8_dequantise_first(enabled: bool) -> None:
    """Lets adr_matmul_nt_fp16u8 dequantise the weight matrix once into a buffer of the pool and
    run the fp16 kernels on it where that is faster (off by default: always the fused kernels)."""
    _ffi.lib().adr_set_u8_dequantise_first(1 if enabled else 0)


class MatmulTracer(CommonKernels):
    """Decorator recording the set of (left, right, output) layouts seen by the matmuls, then
    forwarding (kernels.rs:231-359)."""

    def __init__(self, inner: CommonKernels):
        self.inner = inner
        self._lock = threading.Lock()
        self.shapes = set()

    def clear(self):
        with self._lock:
            self.shapes.clear()

    def _record(self, output, left, right):
        with self._lock:
            self.shapes.add((left.layout, right.layout, output.layout))

    def matmul_f16(self, output, left, right, options=MatmulOptions()):
        self._record(output, left, right)
        self.inner.matmul_f16(output, left, right, options)

    def matmul_f16_slow(self, output, left, right, options=MatmulOptions()):
        self._record(output, left, right)
        self.inner.matmul_f16_slow(output, left, right, options)

    def softmax_rows_inplace(self, output, temperature: float = 1.0):
        self.inner.softmax_rows_inplace(output, temperature)   # forwarded (kernels.rs:334-338)

    def attention_f16(self, output, query, key, value, scale, temperature=1.0,
                      mask=MatmulMask.NONE):
        self.inner.attention_f16(output, query, key, value, scale, temperature, mask)

    def rotary_f16(self, output, input, positions, rotary):
        self.inner.rotary_f16(output, input, positions, rotary)

    def append_f16(self, cache, batch, key, value, rotary=None, query_out=None, query=None, positions=None):
        self.inner.append_f16(cache, batch, key, value, rotary, query_out, query, positions)

    def attention_paged_f16(self, output, query, cache, batch, scale, temperature=1.0, mask=MatmulMask.CAUSAL):
        self.inner.attention_paged_f16(output, query, cache, batch, scale, temperature, mask)

    def attention_packed_f16(self, output, query, key, value, batch, scale, temperature=1.0, mask=MatmulMask.CAUSAL):
        self.inner.attention_packed_f16(output, query, key, value, batch, scale, temperature, mask)

    def error_stats_f16(self, output, lhs, rhs):
        self.inner.error_stats_f16(output, lhs, rhs)            # forwarded (kernels.rs:349-358)

    def error_stats_f32(self, output, lhs, rhs):
        self.inner.error_stats_f32(output, lhs, rhs)
