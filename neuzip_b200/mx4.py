"""Backend that holds tensors in microscaled 4-bit floating point (MXFP4) and multiplies by
them as they are: the counterpart of :class:`neuzip_b200.backend.CodecBackend` with the same
methods, over the ``nz_mx4_*`` calls of ``libneuzip_b200.so``.

Every 32 consecutive elements of the last dimension share a power of two; an element keeps a
sign, two exponent bits and one mantissa bit, 4.25 bits in all.  That holds for matrices with a multiple
of 128 rows and of 256 columns: every matrix is stored in tiles of 128 rows, columns in blocks of 32
with scales for 256 at a time, all filled up.  Low or narrow tensors take more (128 x 32 6 bits an
element, matrices of 16 rows eight times their share, a vector of 4096 elements 544 bits an element);
`size` counts it all.  `linear` and
`grouped_linear` quantise their inputs by the same rule, so that the tensor cores multiply
4-bit operands directly; the weights are never decoded.  The reference has no such form: its
lossy precisions (cuda/kernels.cuh:53-156) keep entropy-coded exponents and decompress before
every product (cuda/high_level.cu:252-263).
"""
from __future__ import annotations

import functools
import math
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence

import torch
from torch.autograd import forward_ad

from . import _lib
from .backend import _ptr

_DTYPES = {torch.bfloat16: _lib.NZ_DTYPE_BF16, torch.float16: _lib.NZ_DTYPE_FP16}
_NAMES = {torch.bfloat16: "bfloat16", torch.float16: "float16"}


@dataclass
class _Entry:
    shape: torch.Size
    dtype: torch.dtype
    matrices: int             # the stack that is stored: [matrices, rows, cols]
    rows: int
    cols: int
    packed: torch.Tensor      # uint8: codes and scales in the tensor cores' order
    streams: set              # streams whose use the allocator knows of
    device: torch.device = field(init=False)

    def __post_init__(self) -> None:
        self.device = self.packed.device

    @property
    def numel(self) -> int:
        return self.matrices * self.rows * self.cols


_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device


class _Here:
    """Nothing to do: the device is the current one already."""

    def __enter__(self):
        pass

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _on(device: torch.device):
    return _HERE if device.index == _current_device() else torch.cuda.device(device)


def _stack(shape: Sequence[int]):
    """How a tensor is stored: three dimensions are a stack of matrices, anything else rows."""
    if len(shape) == 0:
        return 1, 1, 1
    if len(shape) == 3:
        return int(shape[0]), int(shape[1]), int(shape[2])
    return 1, math.prod(int(d) for d in shape[:-1]), int(shape[-1])


@functools.lru_cache(maxsize=512)
def _stored_bytes(matrices: int, rows: int, cols: int) -> int:
    return int(_lib.load().nz_mx4_bytes(matrices, rows, cols))


@functools.lru_cache(maxsize=2048)
def _workspace_bytes(device: int, matrices: int, rows: int, cols: int, n_rows: int, grouped: bool) -> int:
    return int(_lib.load().nz_mx4_linear_workspace_bytes(matrices, rows, cols, n_rows, grouped))


def _has_tangent(tensor: Optional[torch.Tensor]) -> bool:
    return tensor is not None and forward_ad.unpack_dual(tensor).tangent is not None


def _in_autocast_type(tensor: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """What ``functional.linear`` makes of an argument under autocast."""
    if tensor is None or not tensor.is_floating_point() or tensor.dtype == torch.float64:
        return tensor
    return tensor.to(torch.get_autocast_dtype("cuda"))


class _TrainedBias(torch.autograd.Function):
    """A product of inputs that need no gradient and a frozen matrix, whose bias is trained: the bias is
    still added before the one rounding."""

    @staticmethod
    def forward(ctx, bias, product, entry, x, input):
        ctx.shape = bias.shape
        return product(entry, x, input, bias)

    @staticmethod
    def backward(ctx, grad_output):
        return grad_output.reshape(-1, grad_output.shape[-1]).sum(0).reshape(ctx.shape), None, None, None, None


class MX4Backend:
    """`read / write / size / linear / linear_without_bias / split` and the extras of the codec
    backends, on 4-bit storage."""

    supports_operand_order = False
    multiplies_stored = True           # `linear` never decodes: there is nothing to decode ahead

    def __init__(self) -> None:
        self._lib = _lib.load()
        self._cache: Dict[str, _Entry] = {}
        self._status: Dict[int, torch.Tensor] = {}
        self._captured: Dict[int, torch.Tensor] = {}     # bytes that a captured graph reads

    # -- helpers ---------------------------------------------------------
    def _status_of(self, device: int) -> torch.Tensor:
        word = self._status.get(device)
        if word is None:
            if torch._C._cuda_isCurrentStreamCapturing():
                # a word made here would be the graph's: without a value before the first replay, and cleared
                # by every one
                raise RuntimeError("a manager's first product or row lookup on a device cannot be captured in a "
                                   "CUDA graph: make one before the capture")
            _lib.check(self._lib.nz_device_check())
            word = torch.zeros(1, dtype=torch.int32, device=f"cuda:{device}")
            # cleared before any stream may set it; where two threads come first together, one word stays
            torch.cuda.current_stream(device).synchronize()
            word = self._status.setdefault(device, word)
        return word

    def status(self) -> int:
        """Status word accumulated so far, over all devices (synchronises)."""
        bits = 0
        for word in list(self._status.values()):
            bits |= int(word.item()) & 0xFFFFFFFF
        return bits

    def check(self) -> None:
        word = self.status()
        if word:
            raise _lib.NeuzipError("a kernel reported: " + _lib.describe_status(word))

    def _get(self, name: str) -> _Entry:
        entry = self._cache.get(name)
        if entry is None:
            raise RuntimeError("Data not found")
        return entry

    def _use(self, entry: _Entry) -> int:
        """The current stream of the current device, which must be the entry's; from now on
        the allocator does not hand the entry's memory out while that stream may read it."""
        stream = torch._C._cuda_getCurrentRawStream(entry.device.index)
        if torch._C._cuda_isCurrentStreamCapturing():
            # the graph reads these bytes at every replay, whatever becomes of the handle; its end is not
            # known here, see release_captured
            self._captured[entry.packed.data_ptr()] = entry.packed
        if stream not in entry.streams:
            current = torch.cuda.current_stream(entry.device)
            entry.packed.record_stream(current)
            entry.streams.add(stream)
        return stream

    def captured_bytes(self) -> int:
        """Stored bytes that are kept for captured graphs alone: their handle has been written
        again or erased since.  `size` does not count them."""
        held = {entry.packed.data_ptr() for entry in self._cache.values()}
        return sum(packed.numel() for at, packed in self._captured.items() if at not in held)

    def release_captured(self) -> None:
        """Keep nothing more for the graphs that have been captured so far: those that read a handle
        must not be replayed after it is written again or erased.  Waits for the work under way, so
        not inside a capture."""
        if torch.cuda.is_initialized() and torch._C._cuda_isCurrentStreamCapturing():
            raise RuntimeError("release_captured cannot be called inside the capture of a CUDA graph")
        for device in {packed.device for packed in self._captured.values() if packed.is_cuda}:
            torch.cuda.synchronize(device)
        self._captured.clear()

    # -- the six methods of the extension class ----------------------------
    def write(self, name: str, tensor: torch.Tensor) -> None:
        """Quantise `tensor` (bf16 or fp16, any shape; three dimensions are a stack of matrices)
        and keep it under `name`, on its own device (a CPU tensor goes to the current one)."""
        if tensor.dtype not in _DTYPES:
            raise RuntimeError("Unsupported data type")
        if not tensor.is_cuda:
            tensor = tensor.cuda()
        source = tensor if tensor.is_contiguous() else tensor.detach().contiguous()
        with _on(source.device):
            device = source.get_device()
            if device not in self._status and not torch._C._cuda_isCurrentStreamCapturing():
                self._status_of(device)
            shape = source.shape
            matrices, rows, cols = _stack(shape)
            packed = torch.empty(_stored_bytes(matrices, rows, cols), dtype=torch.uint8, device=source.device)
            stream = torch._C._cuda_getCurrentRawStream(device)
            rc = self._lib.nz_mx4_quantize(source.data_ptr(), _DTYPES[source.dtype], matrices, rows, cols,
                                           packed.data_ptr(), stream)
            if rc:
                _lib.check(rc)
        self._cache[name] = _Entry(shape, source.dtype, matrices, rows, cols, packed, {stream})

    def read(self, name: str) -> torch.Tensor:
        """The stored numbers as a flat tensor of the type that was written."""
        entry = self._get(name)
        return self.read_shaped(name, (entry.numel,))

    def read_shaped(self, name: str, shape) -> torch.Tensor:
        """`read` into a tensor of the given shape (one size may be -1)."""
        entry = self._get(name)
        with _on(entry.device):
            if shape == entry.shape:
                out = torch.empty(shape, dtype=entry.dtype, device=entry.device)
            else:
                out = torch.empty(entry.numel, dtype=entry.dtype, device=entry.device).view(tuple(shape))
            rc = self._lib.nz_mx4_dequantize(entry.packed.data_ptr(), entry.matrices, entry.rows, entry.cols,
                                             _DTYPES[entry.dtype], out.data_ptr(), self._use(entry))
            if rc:
                _lib.check(rc)
        return out

    def read_many(self, names: Sequence[str]) -> List[torch.Tensor]:
        return [self.read(name) for name in names]

    def read_rows(self, name: str, rows: torch.Tensor, row_len: int) -> torch.Tensor:
        """Rows ``rows`` (any integer tensor) of the stored tensor seen as a
        ``[numel / row_len, row_len]`` table.  A row outside the table reads as zeros and raises
        at the next ``check()``."""
        entry = self._get(name)
        if row_len <= 0 or entry.numel % row_len:
            raise ValueError(f"row length {row_len} does not divide the {entry.numel} stored elements")
        if rows.is_floating_point() or rows.is_complex() or rows.dtype == torch.bool:
            raise TypeError(f"row numbers must be integers, got {rows.dtype}")
        device = entry.device
        rows = rows.reshape(-1).to(device=device, dtype=torch.int64).contiguous()
        if row_len != entry.cols:
            # rows of several dimensions: each is a run of the table's own rows
            if row_len % entry.cols:
                raise ValueError(f"row length {row_len} is not a whole number of stored rows")
            run = row_len // entry.cols
            rows = rows.clamp(-1, entry.numel // row_len)     # far numbers times `run` could wrap into the table
            rows = (rows.unsqueeze(1) * run + torch.arange(run, device=device)).reshape(-1)
        with _on(device):
            out = torch.empty(rows.numel(), entry.cols, dtype=entry.dtype, device=device)
            _lib.check(self._lib.nz_mx4_gather_rows(
                _ptr(entry.packed), entry.matrices, entry.rows, entry.cols,
                _DTYPES[entry.dtype], _ptr(rows), rows.numel(), _ptr(out),
                _ptr(self._status_of(device.index)), self._use(entry)))
        return out.view(-1, row_len)

    def size(self, name: str) -> int:
        """Stored bytes, 0 for an unknown name."""
        entry = self._cache.get(name)
        return 0 if entry is None else entry.packed.numel()

    def linear(self, name: str, input: torch.Tensor, shape: Sequence[int],
               bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``q(input) @ q(W)^T (+ bias)``: the inputs are quantised like the weights, sums are
        fp32, the result is rounded once to the type of `input` (under autocast, of autocast).
        Differentiable in `bias` alone; inputs that need a gradient are refused (``nn.Linear``
        takes them)."""
        entry = self._get(name)
        if len(shape) != 2 or entry.matrices != 1 or shape[1] != entry.cols or shape[0] != entry.rows:
            raise ValueError(f"linear needs a matrix, got a tensor of shape {tuple(shape)}")
        if torch.is_autocast_enabled():
            input, bias = _in_autocast_type(input), _in_autocast_type(bias)
        x = self._checked_input(entry, input, bias, False)
        if bias is not None and bias.requires_grad and torch.is_grad_enabled():
            return _TrainedBias.apply(bias, self._dense, entry, x, input)
        return self._dense(entry, x, input, bias)

    def _dense(self, entry: _Entry, x: torch.Tensor, input: torch.Tensor,
               bias: Optional[torch.Tensor]) -> torch.Tensor:
        n = x.size(0)
        y = input.new_empty((n, entry.rows) if input.dim() == 2 else (*input.shape[:-1], entry.rows))
        return self._launch(entry, x, n, 1, None, bias, y)

    def linear_without_bias(self, name: str, input: torch.Tensor, shape: Sequence[int]) -> torch.Tensor:
        return self.linear(name, input, shape)

    def grouped_linear(self, name: str, input: torch.Tensor, experts: torch.Tensor,
                       bias: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Row ``r`` of the result is ``q(input[r]) @ q(W[experts[r]])^T (+ bias[experts[r]])`` for a
        stack ``W`` of matrices.  `experts` is an integer tensor; `input` has its shape and one
        more dimension, or lacks its last one, and then every input row goes to all the
        experts named for it (`bias` is ``[E, out]``): ``[T, k]`` experts and ``[T, in]`` inputs give ``[T, k, out]``.
        -1 means no expert and gives a row of zeros; other numbers outside the stack too, and
        they raise at the next ``check()``.  Nothing synchronises with the host."""
        entry = self._get(name)
        if len(entry.shape) != 3:
            raise ValueError("grouped_linear needs a stack of matrices (three dimensions), "
                             f"got a tensor of shape {tuple(entry.shape)}")
        if experts.is_floating_point() or experts.is_complex() or experts.dtype == torch.bool:
            raise TypeError(f"expert numbers must be integers, got {experts.dtype}")
        if experts.device != entry.device:
            raise ValueError(f"expert numbers are on {experts.device}, the weights on {entry.device}")
        lead, per_input = input.shape[:-1], 1
        if lead != experts.shape:
            if experts.dim() == 0 or lead != experts.shape[:-1]:
                raise ValueError(f"inputs of shape {tuple(input.shape)} do not match experts of shape "
                                 f"{tuple(experts.shape)}")
            per_input = int(experts.shape[-1])
        if torch.is_autocast_enabled():
            input, bias = _in_autocast_type(input), _in_autocast_type(bias)
        x = self._checked_input(entry, input, bias, True)
        if bias is not None and bias.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("grouped_linear has no gradient for its bias: detach it, or call under "
                               "torch.no_grad()")
        ids = (experts if experts.dtype == torch.int64 else experts.long()).contiguous()
        y = input.new_empty((*experts.shape, entry.rows))
        return self._launch(entry, x, ids.numel(), per_input, ids, bias, y)

    def _checked_input(self, entry: _Entry, input: torch.Tensor,
                       bias: Optional[torch.Tensor], stack: bool) -> torch.Tensor:
        """`input` as rows one element apart inside, after the checks the products share."""
        if input.dtype not in _DTYPES:
            raise RuntimeError("Unsupported data type")
        shape = input.shape
        if not shape or shape[-1] != entry.cols or entry.cols == 0:
            raise ValueError(f"inputs of shape {tuple(shape)} do not fit weights of shape "
                             f"{tuple(entry.shape)}")
        if input.device != entry.device:
            raise ValueError(f"inputs are on {input.device}, the weights on {entry.device}")
        if bias is not None:
            if bias.dtype != input.dtype or bias.device != entry.device:
                raise ValueError(f"bias must be of type {_NAMES[input.dtype]} on {entry.device}, got "
                                 f"{bias.dtype} on {bias.device}")
            # a vector's numbers have one order whatever its shape, those of a stack do not
            if bias.shape != (entry.matrices, entry.rows) if stack else bias.numel() != entry.rows:
                raise ValueError(f"bias must have the shape {(entry.matrices, entry.rows) if stack else (entry.rows,)}, "
                                 f"got {tuple(bias.shape)}")
        if input.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("a manager's products with 4-bit weights have no gradient for their inputs: use "
                               "nn.Linear for one matrix, or call under torch.no_grad()")
        # outside every dual_level there is nothing to unpack (which takes 0.4 us)
        if getattr(forward_ad, "_current_level", 0) >= 0 and (_has_tangent(input) or _has_tangent(bias)):
            raise NotImplementedError("products with 4-bit weights have no forward-mode derivative")
        x = input if len(shape) == 2 else input.reshape(-1, entry.cols)
        row, element = x.stride()
        if element != 1 or row < entry.cols:
            x = x.contiguous()
        return x

    def _launch(self, entry: _Entry, x: torch.Tensor, n_rows: int, per_input: int,
                ids: Optional[torch.Tensor], bias: Optional[torch.Tensor], y: torch.Tensor) -> torch.Tensor:
        if n_rows == 0 or entry.rows == 0:
            return y
        device = entry.device.index
        if device != _current_device():
            with torch.cuda.device(device):
                return self._launch(entry, x, n_rows, per_input, ids, bias, y)
        need = _workspace_bytes(device, entry.matrices, entry.rows, entry.cols, n_rows, ids is not None)
        # from the allocator on every call: calls on other streams and captured graphs have their own
        workspace = x.new_empty(need, dtype=torch.uint8) if need else None
        if bias is not None:
            bias = bias.contiguous()
        status = self._status.get(device)
        if status is None:
            status = self._status_of(device)
        rc = self._lib.nz_mx4_linear(
            entry.packed.data_ptr(), entry.matrices, entry.rows, entry.cols, _DTYPES[x.dtype], x.data_ptr(),
            x.stride(0), n_rows, per_input, None if ids is None else ids.data_ptr(),
            None if bias is None else bias.data_ptr(), y.data_ptr(),
            None if workspace is None else workspace.data_ptr(), need, status.data_ptr(), self._use(entry))
        if rc:
            _lib.check(rc)
        return y

    def split(self, tensor: torch.Tensor):
        raise NotImplementedError("4-bit storage has no split()")

    # -- serialisation ----------------------------------------------------
    def export_entry(self, name: str) -> dict:
        """The stored form of one tensor as CPU tensors plus what is needed to read it."""
        e = self._cache[name]
        return {"format": "MXFP4", "dtype": _NAMES[e.dtype], "stack": (e.matrices, e.rows, e.cols),
                "packed": e.packed.cpu()}

    def _import_device(self, name: str, device) -> torch.device:
        """The GPU asked for, else the one that holds `name` already, else the current one."""
        device = None if device is None else torch.device(device)
        if device is None or device.type != "cuda":
            held = self._cache.get(name)
            device = torch.device("cuda") if held is None else held.device
        return device if device.index is not None else torch.device("cuda", torch.cuda.current_device())

    def import_entry(self, name: str, blob: dict, device=None) -> None:
        """Inverse of `export_entry`: the stored bytes go straight to `device`, a GPU; by default to
        the one that holds the entry they replace, or the current one."""
        if blob.get("format") != "MXFP4":
            raise ValueError(f"checkpoint entry does not match this manager (format {blob.get('format')!r})")
        shape = torch.Size(blob["shape"])
        stack = _stack(shape)
        dtype = {v: k for k, v in _NAMES.items()}.get(blob["dtype"])
        if dtype is None or tuple(blob["stack"]) != stack:
            raise ValueError("checkpoint entry: type or shape does not fit the stored bytes")
        if blob["packed"].dtype != torch.uint8 or blob["packed"].numel() != _stored_bytes(*stack):
            raise ValueError("checkpoint entry: the stored bytes have the wrong length")
        device = self._import_device(name, device)
        with _on(device):
            packed = blob["packed"].to(device=device, copy=True).contiguous()
            if not torch._C._cuda_isCurrentStreamCapturing():
                self._status_of(device.index)
            self._cache[name] = _Entry(shape, dtype, *stack, packed,
                                       {torch._C._cuda_getCurrentRawStream(device.index)})

    # -- extras -----------------------------------------------------------
    def erase(self, name: str) -> None:
        self._cache.pop(name, None)

    def entry(self, name: str) -> _Entry:
        return self._cache[name]

    def names(self):
        return list(self._cache)
