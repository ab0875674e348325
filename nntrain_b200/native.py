"""Checked wrappers over the C ABI, one per managed wrapper class of the
reference.  They validate device / dtype / length the way the managed wrappers
do, pass raw device pointers across the boundary, and turn a non-zero status
into NativeCudaError.  Tensors are torch CUDA tensors used purely as device
buffers.

  CudaBfp8Native          NNtrain.Core/Tensors/CudaBfp8Native.cs (QuantizeFloat32, ...)
  CudaBfp8GradientNative  NNtrain.Core/Tensors/CudaBfp8GradientNative.cs:10-237
  CudaGradientBuckets     NNtrain.Core/Tensors/CudaGradientBuckets.cs:6-349
  GradientNorm            the norm / clip kernels behind
                          NNtrain.Core/Tensors/Tensor.CudaKernels.cs:119-854
  RmsNorm                 root-mean-square norm with an encoded output, and its gradient
  TokenEmbedding          rows of a (possibly encoded) token table, and the table's gradient
  GradientTensorList      the leaves that clip_grad_norm_ walks there, as one
                          table (NNtrain.Core/Torch/nn.cs:32-81)
"""
from __future__ import annotations

import ctypes
import functools
import itertools

import numpy as np
import torch

from .library import check, load


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _stream(stream) -> int:
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _require(t: torch.Tensor, dtype, name: str, device: int | None = None) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if device is not None and t.device.index != device:
        raise ValueError(f"{name} is on device {t.device.index}, expected {device}")


_F32 = torch.float32
_FLOAT32, _BFLOAT16 = (torch.float32,), (torch.bfloat16, torch.int16)   # bf16 values, or their bits
_FLOATS = _FLOAT32 + _BFLOAT16
_INT32, _INT8, _INTEGERS = (torch.int32,), (torch.int8,), (torch.int64, torch.int32)
_current_raw_stream = torch._C._cuda_getCurrentRawStream


def _kind(t: torch.Tensor) -> int:
    """0 = fp32, 1 = bf16 (the kinds of the C boundary)."""
    return 0 if t.dtype is _F32 else 1


def _stream_on(device: int, stream) -> int:
    """The handle of `stream`, or of the device's current stream."""
    if stream is None:
        return _current_raw_stream(device)
    return stream if isinstance(stream, int) else stream.cuda_stream


def _scratch(device: int, bytes_: int, stream):
    """Device scratch for one call on `stream`.  It is allocated on that stream,
    so it is not handed out again before the call's kernels have run."""
    if bytes_ == 0:
        return None
    if stream is None:
        return torch.empty(bytes_, dtype=torch.uint8, device=torch.device("cuda", device))
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(bytes_, dtype=torch.uint8, device=torch.device("cuda", device))


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(function: str, *sizes) -> int:
    """What the library's host-only function says that a call of these sizes needs."""
    need = ctypes.c_longlong()
    check(function, getattr(load(), function)(*sizes, ctypes.addressof(need)))
    return need.value


def _workspace(function: str, sizes, device: int, given, stream):
    """(scratch, its bytes) for one call: the caller's, or allocated for it."""
    need = _scratch_bytes(function, *sizes)
    if given is None:
        return _scratch(device, need, stream), need
    _require(given, torch.uint8, "workspace", device)
    if given.numel() < need:
        raise ValueError(f"workspace has {given.numel()} bytes, needs {need}")
    return given, given.numel()


def _vector(t: torch.Tensor, name: str, device: int, length: int, dtypes) -> int:
    """Checks a contiguous tensor of `length` values and returns its address."""
    if not (t.dtype in dtypes and t.numel() == length and t.get_device() == device and t.is_contiguous()):
        _require(t, t.dtype, name, device)
        if t.dtype not in dtypes:
            raise ValueError(f"{name} has type {t.dtype}, expected one of {', '.join(map(str, dtypes))}")
        raise ValueError(f"{name} has {t.numel()} values, expected {length}")
    return t.data_ptr()


def _status(t, name: str, device: int) -> int:
    """Checks an optional int32 flag and returns its address."""
    if t is None:
        return 0
    if t.numel() < 1:
        raise ValueError(f"{name} needs a value")
    return _vector(t, name, device, t.numel(), _INT32)


def _rows(t: torch.Tensor, name: str, device: int, width: int, dtypes, rows: int | None = None) -> int:
    """Checks a matrix of rows (contiguous values, any row stride) and returns the stride."""
    if t.get_device() != device:
        raise ValueError(f"{name} must be on CUDA device {device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} has type {t.dtype}, expected one of {', '.join(map(str, dtypes))}")
    shape = t.shape
    if len(shape) != 2 or shape[1] != width or (rows is not None and shape[0] != rows):
        raise ValueError(f"{name} has shape {tuple(shape)}, expected ({'rows' if rows is None else rows}, {width})")
    row, value = t.stride()
    if value != 1 and width > 1 and shape[0] > 0:
        raise ValueError(f"{name}: the values of a row must be contiguous")
    if shape[0] <= 1:
        return width
    if row < width:
        raise ValueError(f"{name}: rows must not overlap")
    return row


def scale_count(length: int, block_size: int) -> int:
    """Bfp8QuantizationDescriptor.GetScaleCount
    (NNtrain.Core/Tensors/Bfp8Quantization.cs:64-78); block_size 0 = tensor-wide."""
    block = max(1, length) if block_size <= 0 or block_size >= length else block_size
    return (length + block - 1) // block


class CudaBfp8Native:
    """Block / tensor-wide codec.  block_size 0 means tensor-wide."""

    @staticmethod
    def quantize_float32(device: int, source, payload, scales, block_size: int, stream=None) -> None:
        _require(source, torch.float32, "source", device)
        _require(payload, torch.int8, "payload", device)
        _require(scales, torch.float32, "scales", device)
        n = source.numel()
        if payload.numel() != n or scales.numel() != scale_count(n, block_size):
            raise ValueError("BFP8 payload / scale lengths do not match the descriptor")
        block = n if block_size <= 0 else block_size
        check("bfp8_quantize_f32", load().nntrain_cuda_bfp8_quantize_f32(
            device, _ptr(source), _ptr(payload), _ptr(scales), n, block, _stream(stream)))

    @staticmethod
    def dequantize_float32(device: int, payload, scales, destination, block_size: int, stream=None) -> None:
        _require(payload, torch.int8, "payload", device)
        _require(scales, torch.float32, "scales", device)
        _require(destination, torch.float32, "destination", device)
        n = payload.numel()
        if destination.numel() != n or scales.numel() != scale_count(n, block_size):
            raise ValueError("BFP8 payload / scale lengths do not match the descriptor")
        block = n if block_size <= 0 else block_size
        check("bfp8_dequantize_f32", load().nntrain_cuda_bfp8_dequantize_f32(
            device, _ptr(payload), _ptr(scales), _ptr(destination), n, block, _stream(stream)))

    @staticmethod
    def quantize_bfloat16(device: int, source_bits, payload, scales, block_size: int, stream=None) -> None:
        """`source_bits`: bf16 bit patterns (int16 tensor)."""
        _require(source_bits, torch.int16, "source", device)
        _require(payload, torch.int8, "payload", device)
        n = source_bits.numel()
        if payload.numel() != n or scales.numel() != scale_count(n, block_size):
            raise ValueError("BFP8 payload / scale lengths do not match the descriptor")
        check("cuda_bfp8_quantize_bf16", load().nntrain_cuda_bfp8_quantize_bf16(
            device, _ptr(source_bits), _ptr(payload), _ptr(scales), n, n if block_size <= 0 else block_size,
            _stream(stream)))

    @staticmethod
    def dequantize_bfloat16(device: int, payload, scales, destination_bits, block_size: int, stream=None) -> None:
        _require(destination_bits, torch.int16, "destination", device)
        n = payload.numel()
        if destination_bits.numel() != n or scales.numel() != scale_count(n, block_size):
            raise ValueError("BFP8 payload / scale lengths do not match the descriptor")
        check("cuda_bfp8_dequantize_bf16", load().nntrain_cuda_bfp8_dequantize_bf16(
            device, _ptr(payload), _ptr(scales), _ptr(destination_bits), n, n if block_size <= 0 else block_size,
            _stream(stream)))

    @staticmethod
    def quantize_float32_roundtrip(device: int, state, payload, scales, block_size: int, stream=None) -> None:
        _require(state, torch.float32, "state", device)
        _require(payload, torch.int8, "payload", device)
        _require(scales, torch.float32, "scales", device)
        n = state.numel()
        check("bfp8_quantize_f32_roundtrip", load().nntrain_cuda_bfp8_quantize_f32_roundtrip(
            device, _ptr(state), _ptr(payload), _ptr(scales), n, block_size, _stream(stream)))

    @staticmethod
    def block_encode(device: int, source, payload, scales, block_size: int, roundtrip=None,
                     squared_sum=None, finite_status=None, stream=None) -> None:
        """64-bit-length encode with optional fused write-back / sum of squares / finite flag."""
        _require(source, torch.float32, "source", device)
        _require(payload, torch.int8, "payload", device)
        _require(scales, torch.float32, "scales", device)
        n = source.numel()
        if payload.numel() < n or scales.numel() < scale_count(n, block_size):
            raise ValueError("BFP8 payload / scale buffers are too small")
        check("bfp8_block_encode", load().nntrain_bfp8_block_encode(
            device, _ptr(source), _ptr(payload), _ptr(scales), n, block_size, _ptr(roundtrip),
            _ptr(squared_sum), _ptr(finite_status), _stream(stream)))

    @staticmethod
    def block_decode(device: int, payload, scales, destination, block_size: int, stream=None) -> None:
        _require(payload, torch.int8, "payload", device)
        _require(destination, torch.float32, "destination", device)
        n = destination.numel()
        check("bfp8_block_decode", load().nntrain_bfp8_block_decode(
            device, _ptr(payload), _ptr(scales), _ptr(destination), n, block_size, _stream(stream)))


class CudaBfp8GradientNative:
    """Tensor-wide gradient publication and the 2-device reduce / broadcast."""

    @staticmethod
    def quantize(device: int, gradient, payload, scale, finite_status, squared_sum=None, stream=None) -> None:
        _require(gradient, torch.float32, "gradient", device)
        _require(payload, torch.int8, "payload", device)
        _require(scale, torch.float32, "scale", device)
        _require(finite_status, torch.int32, "finite_status", device)
        n = gradient.numel()
        if payload.numel() != n or scale.numel() != 1:
            raise ValueError("tensor-wide BFP8 gradient needs numel payload bytes and one scale")
        lib = load()
        if squared_sum is None:
            check("bfp8_gradient_quantize", lib.nntrain_bfp8_gradient_quantize(
                device, _ptr(gradient), _ptr(payload), _ptr(scale), n, _ptr(finite_status), _stream(stream)))
        else:
            _require(squared_sum, torch.float64, "squared_sum", device)
            check("bfp8_gradient_quantize_accumulate", lib.nntrain_bfp8_gradient_quantize_accumulate(
                device, _ptr(gradient), _ptr(payload), _ptr(scale), n, _ptr(finite_status),
                _ptr(squared_sum), _stream(stream)))

    @staticmethod
    def publish_tensors(device: int, arena, payload, scales, tensor_offsets, maxima_scratch, finite_status,
                        squared_sum=None, stream=None) -> None:
        """Every tensor of a bucket arena in three stream operations:
        `tensor_offsets` is a device int64 tensor of tensors + 1 ascending
        element offsets, `scales` / `maxima_scratch` have one entry per tensor."""
        _require(arena, torch.float32, "arena", device)
        _require(payload, torch.int8, "payload", device)
        _require(scales, torch.float32, "scales", device)
        _require(tensor_offsets, torch.int64, "tensor_offsets", device)
        _require(maxima_scratch, torch.int32, "maxima_scratch", device)
        tensors = tensor_offsets.numel() - 1
        if payload.numel() != arena.numel() or scales.numel() != tensors or maxima_scratch.numel() < tensors:
            raise ValueError("payload / scales / scratch sizes do not match the arena and the offset table")
        check("bfp8_gradient_publish_tensors", load().nntrain_bfp8_gradient_publish_tensors(
            device, _ptr(arena), _ptr(payload), _ptr(scales), _ptr(tensor_offsets), tensors, arena.numel(),
            _ptr(maxima_scratch), _ptr(finite_status), _ptr(squared_sum), _stream(stream)))

    @staticmethod
    def reduce_tensors(device: int, payloads, scales, reduced, out_payload, out_scales, tensor_offsets,
                       maxima_scratch, finite_status, reduction_scale: float = 1.0, squared_sum=None,
                       stream=None) -> None:
        import ctypes
        tensors = tensor_offsets.numel() - 1
        table_p = (ctypes.c_void_p * len(payloads))(*[_ptr(p) for p in payloads])
        table_s = (ctypes.c_void_p * len(scales))(*[_ptr(s) for s in scales])
        check("bfp8_gradient_reduce_tensors", load().nntrain_bfp8_gradient_reduce_tensors(
            device, len(payloads), table_p, table_s, _ptr(reduced), _ptr(out_payload), _ptr(out_scales),
            _ptr(tensor_offsets), tensors, reduced.numel(), reduction_scale, _ptr(maxima_scratch),
            _ptr(finite_status), _ptr(squared_sum), _stream(stream)))

    @staticmethod
    def decode_tensors(device: int, payload, scales, destination, tensor_offsets, skip_flag=None,
                       stream=None) -> None:
        check("bfp8_gradient_decode_tensors", load().nntrain_bfp8_gradient_decode_tensors(
            device, _ptr(payload), _ptr(scales), _ptr(destination), _ptr(tensor_offsets),
            tensor_offsets.numel() - 1, destination.numel(), _ptr(skip_flag), _stream(stream)))

    @staticmethod
    def accumulate_squared_sum(device: int, payload, scale, squared_sum, finite_status, stream=None) -> None:
        check("bfp8_gradient_squared_sum", load().nntrain_bfp8_gradient_squared_sum(
            device, _ptr(payload), _ptr(scale), payload.numel(), _ptr(squared_sum), _ptr(finite_status),
            _stream(stream)))

    @staticmethod
    def scale(device: int, scale, multiplier: float, stream=None) -> None:
        check("bfp8_gradient_scale", load().nntrain_bfp8_gradient_scale(
            device, _ptr(scale), multiplier, _stream(stream)))

    @staticmethod
    def reduce(primary: int, secondary: int, local_payload, local_scale, remote_payload, remote_scale,
               remote_payload_staging, remote_scale_staging, reduced, output_payload, output_scale,
               reduction_scale: float, finite_status, remote_finite_status, remote_status_staging,
               squared_sum, communication_stream: int, local_ready: int, remote_ready: int,
               reduced_ready: int) -> None:
        check("bfp8_gradient_reduce", load().nntrain_bfp8_gradient_reduce(
            primary, secondary, _ptr(local_payload), _ptr(local_scale), _ptr(remote_payload),
            _ptr(remote_scale), _ptr(remote_payload_staging), _ptr(remote_scale_staging), _ptr(reduced),
            _ptr(output_payload), _ptr(output_scale), reduced.numel(), reduction_scale,
            _ptr(finite_status), _ptr(remote_finite_status), _ptr(remote_status_staging),
            _ptr(squared_sum), communication_stream, local_ready, remote_ready, reduced_ready))

    @staticmethod
    def broadcast(destination: int, source: int, source_payload, source_scale, destination_payload,
                  destination_scale, destination_float, destination_finite_status,
                  destination_stream: int, source_ready: int) -> None:
        check("bfp8_gradient_broadcast", load().nntrain_bfp8_gradient_broadcast(
            destination, source, _ptr(source_payload), _ptr(source_scale), _ptr(destination_payload),
            _ptr(destination_scale), _ptr(destination_float), destination_float.numel(),
            _ptr(destination_finite_status), destination_stream, source_ready))


class CudaGradientBuckets:
    """Bucket transport between two devices of one process."""

    @staticmethod
    def create_communication_stream(device: int) -> int:
        import ctypes
        handle = ctypes.c_void_p()
        with torch.cuda.device(device):
            check("gradient_comm_create", load().nntrain_gradient_comm_create(device, ctypes.addressof(handle)))
        return handle.value

    @staticmethod
    def create_ready_event(device: int) -> int:
        import ctypes
        handle = ctypes.c_void_p()
        with torch.cuda.device(device):
            check("gradient_event_create", load().nntrain_gradient_event_create(device, ctypes.addressof(handle)))
        return handle.value

    @staticmethod
    def pack(device: int, source, destination_bf16, destination_offset: int, stream=None) -> None:
        _require(source, torch.float32, "source", device)
        check("gradient_pack_bf16", load().nntrain_gradient_pack_bf16(
            device, _ptr(source), _ptr(destination_bf16), destination_offset, source.numel(), _stream(stream)))

    @staticmethod
    def pack_bfp8_block(device: int, source, destination, scales, stream=None) -> None:
        _require(source, torch.float32, "source", device)
        _require(destination, torch.int8, "destination", device)
        check("gradient_pack_bfp8_block", load().nntrain_gradient_pack_bfp8_block(
            device, _ptr(source), _ptr(destination), _ptr(scales), source.numel(), _stream(stream)))

    @staticmethod
    def record_ready(device: int, event: int, stream=None, external: bool = False) -> None:
        fn = load().nntrain_gradient_record_ready_external if external else load().nntrain_gradient_record_ready
        check("gradient_record_ready", fn(device, event, _stream(stream)))

    @staticmethod
    def exchange(destination_device: int, source_device: int, local, remote_source, remote_staging, reduced,
                 squared_sum, communication_stream: int, local_ready: int, remote_ready: int) -> None:
        check("gradient_exchange_bf16", load().nntrain_gradient_exchange_bf16(
            destination_device, source_device, _ptr(local), _ptr(remote_source), _ptr(remote_staging),
            _ptr(reduced), reduced.numel(), _ptr(squared_sum), communication_stream, local_ready, remote_ready))

    @staticmethod
    def exchange_bfp8_block(destination_device: int, source_device: int, local, local_scales, remote_source,
                            remote_source_scales, remote_staging, remote_staging_scales, reduced, squared_sum,
                            communication_stream: int, local_ready: int, remote_ready: int) -> None:
        check("gradient_exchange_bfp8_block", load().nntrain_gradient_exchange_bfp8_block(
            destination_device, source_device, _ptr(local), _ptr(local_scales), _ptr(remote_source),
            _ptr(remote_source_scales), _ptr(remote_staging), _ptr(remote_staging_scales), _ptr(reduced),
            reduced.numel(), _ptr(squared_sum), communication_stream, local_ready, remote_ready))

    @staticmethod
    def create_host_pipeline(source_device: int, destination_device: int, chunk_elements: int,
                             bfp8_block: bool = False) -> int:
        """The pinned-host fallback for a device pair without peer access."""
        import ctypes
        handle = ctypes.c_void_p()
        fn = (load().nntrain_gradient_host_pipeline_create_bfp8_block if bfp8_block
              else load().nntrain_gradient_host_pipeline_create)
        check("gradient_host_pipeline_create", fn(source_device, destination_device, chunk_elements,
                                                  ctypes.addressof(handle)))
        return handle.value

    @staticmethod
    def host_pipeline_exchange(pipeline: int, local, remote_source, reduced, squared_sum, local_ready: int,
                               remote_ready: int) -> None:
        check("gradient_host_pipeline_exchange_bf16", load().nntrain_gradient_host_pipeline_exchange_bf16(
            pipeline, _ptr(local), _ptr(remote_source), _ptr(reduced), reduced.numel(), _ptr(squared_sum),
            local_ready, remote_ready))

    @staticmethod
    def host_pipeline_exchange_bfp8_block(pipeline: int, local, local_scales, remote_source, remote_source_scales,
                                          reduced, squared_sum, local_ready: int, remote_ready: int) -> None:
        check("gradient_host_pipeline_exchange_bfp8_block",
              load().nntrain_gradient_host_pipeline_exchange_bfp8_block(
                  pipeline, _ptr(local), _ptr(local_scales), _ptr(remote_source), _ptr(remote_source_scales),
                  _ptr(reduced), reduced.numel(), _ptr(squared_sum), local_ready, remote_ready))

    @staticmethod
    def destroy_host_pipeline(pipeline: int) -> None:
        check("gradient_host_pipeline_destroy", load().nntrain_gradient_host_pipeline_destroy(pipeline))

    @staticmethod
    def unpack(device: int, source, source_offset: int, destination, communication_stream: int) -> None:
        check("gradient_unpack_float", load().nntrain_gradient_unpack_float(
            device, _ptr(source), source_offset, _ptr(destination), destination.numel(), communication_stream))

    @staticmethod
    def synchronize(device: int, communication_stream: int) -> None:
        check("gradient_comm_synchronize", load().nntrain_gradient_comm_synchronize(device, communication_stream))

    @staticmethod
    def destroy_event(device: int, event: int) -> None:
        check("gradient_event_destroy", load().nntrain_gradient_event_destroy(device, event))

    @staticmethod
    def destroy_communication_stream(device: int, stream: int) -> None:
        check("gradient_comm_destroy", load().nntrain_gradient_comm_destroy(device, stream))


class GradientTensorList:
    """The gradient tensors of a model as one table on the device: fp32, bf16 and
    BFP8 (payload, with its scales and block size) tensors of any length and
    place, each with an optional destination for its clipped values (BFP8: its
    clipped scales); without one it is clipped in place.  What is written for one
    tensor may not be read or written for another.  Build it once for leaves that
    stay where they are; it holds on to the tensors, and a recorded graph needs
    it to live as long as itself.  Otherwise it may be dropped as soon as a call
    has returned; only a call on a stream given by its handle (or as an
    ExternalStream, which may end before the list does) needs it until its
    kernels have run."""

    _TENSOR = np.dtype([("values", np.uint64), ("scales", np.uint64), ("destination", np.uint64),
                        ("length", np.int64), ("first_chunk", np.int64), ("kind", np.int32), ("block_size", np.int32)])

    def __init__(self, device: int, tensors, scales=None, block_sizes=None, destinations=None):
        count = len(tensors)
        scales = [None] * count if scales is None else list(scales)
        block_sizes = [0] * count if block_sizes is None else list(block_sizes)
        destinations = [None] * count if destinations is None else list(destinations)
        if count == 0 or not len(scales) == len(block_sizes) == len(destinations) == count:
            raise ValueError("a gradient list needs tensors, and one scale, block size and destination for each of them")
        rows = []
        for i, (t, s, block, to) in enumerate(zip(tensors, scales, block_sizes, destinations)):
            length, encoded = t.numel(), t.dtype is torch.int8
            if not encoded and t.dtype not in _FLOATS:
                raise ValueError(f"tensor {i} must be float32, bfloat16 or an int8 payload, got {t.dtype}")
            kind = 2 if encoded else _kind(t)
            if t.get_device() != device or not t.is_contiguous():
                _require(t, t.dtype, f"tensor {i}", device)
            if not encoded:
                if s is not None:
                    raise ValueError(f"tensor {i} is not a BFP8 payload: it has no scales")
                scale_address, block, types, written = 0, 0, _BFLOAT16 if kind else _FLOAT32, length
            else:
                if s is None or block < 0:
                    raise ValueError(f"tensor {i} is a BFP8 payload: it needs its scales and block size")
                _require(s, torch.float32, f"scales of tensor {i}", device)
                if length and s.numel() != scale_count(length, block):
                    raise ValueError(f"tensor {i}: payload / scale lengths do not match the descriptor")
                scale_address, types, written = s.data_ptr(), _FLOAT32, s.numel()
            address = 0
            if to is not None:
                if to.dtype not in types:
                    raise ValueError(f"destination of tensor {i} must have its type")
                if to.numel() != written:
                    raise ValueError(f"destination of tensor {i} must have its length")
                address = _vector(to, f"destination of tensor {i}", device, written, types)
            rows.append((t.data_ptr(), scale_address, address, length, 0, kind, block))
        table = np.array(rows, dtype=self._TENSOR)
        chunks, values = ctypes.c_longlong(), ctypes.c_int()
        plan = load().nntrain_gradient_list_plan
        status = plan(table.ctypes.data, count, None, 0, ctypes.addressof(chunks), ctypes.addressof(values))
        if status == 1:                       # types, lengths and addresses were checked above
            raise ValueError("tensors and destinations of a gradient list must not overlap: what is written for one tensor "
                             "may not be read or written for another")
        check("gradient_list_plan", status)
        # table and chunk map in one buffer, one copy
        buffer = np.zeros(table.nbytes + max(chunks.value, 1) * 8, dtype=np.uint8)
        check("gradient_list_plan", plan(table.ctypes.data, count, buffer.ctypes.data + table.nbytes, chunks.value,
                                         ctypes.addressof(chunks), ctypes.addressof(values)))
        buffer[:table.nbytes] = table.view(np.uint8)
        self.device, self.count, self.chunks, self.chunk_values = device, count, chunks.value, values.value
        self.buffer = torch.from_numpy(buffer).to(torch.device("cuda", device))
        self.table_address = self.buffer.data_ptr()
        self.map_address = self.table_address + table.nbytes
        self._held = (list(tensors), scales, destinations)
        self._streams = {_current_raw_stream(device)}

    def _keep_for(self, stream, handle: int) -> None:
        """Table and tensors are not handed out again before what is now on
        `stream`, not the one the list was built on, has run: told to torch's
        allocator once for each stream."""
        if isinstance(stream, (int, torch.cuda.ExternalStream)):
            return
        if stream is None:
            stream = torch.cuda.current_stream(self.device)
        for t in (self.buffer, *itertools.chain(*self._held)):
            if t is not None:
                t.record_stream(stream)
        self._streams.add(handle)


class GradientNorm:
    """Sum of squares and clip kernels (kinds: 0 fp32, 1 bf16, 2 BFP8)."""

    FP32, BF16, BFP8 = 0, 1, 2

    @staticmethod
    def squared_sum(device: int, kind: int, values, squared_sum, scales=None, block_size: int = 0,
                    finite_status=None, stream=None) -> None:
        _require(squared_sum, torch.float64, "squared_sum", device)
        check("gradient_squared_sum", load().nntrain_gradient_squared_sum(
            device, kind, _ptr(values), _ptr(scales), values.numel(), block_size, _ptr(squared_sum),
            _ptr(finite_status), _stream(stream)))

    @staticmethod
    def clip_coefficient(device: int, squared_sum, max_norm: float, norm_and_coefficient, stream=None) -> None:
        check("gradient_clip_coefficient", load().nntrain_gradient_clip_coefficient(
            device, _ptr(squared_sum), max_norm, _ptr(norm_and_coefficient), _stream(stream)))

    @staticmethod
    def clip_apply(device: int, kind: int, values, multiplier: float = 1.0, coefficient=None, stream=None) -> None:
        check("gradient_clip_apply", load().nntrain_gradient_clip_apply(
            device, kind, _ptr(values), values.numel(), multiplier, _ptr(coefficient), _stream(stream)))

    @staticmethod
    def clip_tensors(device: int, tensors: GradientTensorList, max_norm: float, norm_and_coefficient,
                     tensor_norms=None, finite_status=None, apply: bool = True, workspace=None, stream=None) -> None:
        """The global norm over a list and, with `apply`, the clip of every tensor
        of it, without a host read.  `workspace` (optional):
        at least `tensors.chunks` float64 values that no call in flight at the
        same time uses."""
        if tensors.device != device:
            raise ValueError(f"the list is on device {tensors.device}, expected {device}")
        if norm_and_coefficient.numel() < 2:
            raise ValueError("norm_and_coefficient needs two values")
        out = _vector(norm_and_coefficient, "norm_and_coefficient", device, norm_and_coefficient.numel(), _FLOAT32)
        if not max_norm > 0.0:
            raise ValueError("max_norm must be positive")
        norms = 0
        if tensor_norms is not None:
            if tensor_norms.numel() < tensors.count:
                raise ValueError("tensor_norms needs one value for each tensor")
            norms = _vector(tensor_norms, "tensor_norms", device, tensor_norms.numel(), _FLOAT32)
        status = _status(finite_status, "finite_status", device)
        if workspace is None:
            workspace = _scratch(device, tensors.chunks * 8, stream)
        else:
            _require(workspace, torch.float64, "workspace", device)
            if workspace.numel() < tensors.chunks:
                raise ValueError("workspace is too small")
        handle = _stream_on(device, stream)
        if handle not in tensors._streams:
            tensors._keep_for(stream, handle)
        check("gradient_list_clip", load().nntrain_gradient_list_clip(
            device, tensors.table_address, tensors.count, tensors.map_address, tensors.chunks, tensors.chunk_values,
            0 if workspace is None else workspace.data_ptr(), max_norm, apply, out, norms, status, handle))


class Bfp8GradientOptimizers:
    """Optimizer heads that read the reduced BFP8 gradient without a decode pass."""

    @staticmethod
    def adamw(device: int, data, gradient_payload, gradient_scales, block_size: int, first_moment, second_moment,
              beta1: float, beta2: float, learning_rate: float, weight_decay: float, update_scale: float,
              scaled_epsilon: float, apply_weight_decay: bool = True, compute_bf16=None, stream=None) -> None:
        for name, t in (("data", data), ("first_moment", first_moment), ("second_moment", second_moment)):
            _require(t, torch.float32, name, device)
        _require(gradient_payload, torch.int8, "gradient_payload", device)
        n = data.numel()
        if (gradient_payload.numel() != n or first_moment.numel() != n or second_moment.numel() != n
                or gradient_scales.numel() != scale_count(n, block_size)):
            raise ValueError("parameter, moment and gradient sizes do not match")
        check("optimizer_adamw_bfp8_gradient", load().nntrain_optimizer_adamw_bfp8_gradient(
            device, _ptr(data), _ptr(gradient_payload), _ptr(gradient_scales), block_size, _ptr(first_moment),
            _ptr(second_moment), _ptr(compute_bf16), n, beta1, beta2, learning_rate, weight_decay, update_scale,
            scaled_epsilon, int(apply_weight_decay), _stream(stream)))


class RmsNorm:
    """Root-mean-square norm of x + residual whose output goes to the codec's 8
    bits, and its gradient.  Matrices are (rows, width), fp32 or bf16 (bfloat16
    or its bits); inputs may have any row stride, outputs are contiguous."""

    @staticmethod
    def forward(device: int, x, weight, epsilon: float, residual=None, residual_out=None, y=None, payload=None,
                scales=None, block_size: int = 0, inverse_rms=None, finite_status=None, stream=None) -> None:
        """h = x + residual, i = 1 / sqrt(mean(h^2) + epsilon), y = h * i * weight.
        `payload` and `scales`: y encoded, `block_size` values to a scale (a divisor
        of the width; 0 = one scale a row).  `y` (fp32 or bf16): y itself, or with a
        payload the values that the codes stand for.  `residual_out`: h, in x's
        type; `inverse_rms`: i for the gradient.  residual_out, or y in x's type,
        may be x or residual itself."""
        if x.dim() != 2:
            raise ValueError(f"x has shape {tuple(x.shape)}, expected (rows, width)")
        rows, width = x.shape
        kind = _kind(x)
        same = _BFLOAT16 if kind else _FLOAT32
        x_stride = _rows(x, "x", device, width, same)
        weight_address = _vector(weight, "weight", device, width, _FLOATS)
        residual_stride = residual_address = h = inverse = y_address = y_kind = codes = scale_address = 0
        if residual is not None:
            residual_stride, residual_address = _rows(residual, "residual", device, width, same, rows), residual.data_ptr()
        if y is None and payload is None:
            raise ValueError("the norm needs an output: y, or payload and scales")
        if y is not None:
            y_address, y_kind = _vector(y, "y", device, rows * width, _FLOATS), _kind(y)
        if residual_out is not None:
            if residual is None:
                raise ValueError("residual_out without a residual is x itself")
            h = _vector(residual_out, "residual_out", device, rows * width, same)
        if payload is not None:
            block = width if block_size == 0 or block_size > width else block_size
            if block < 0 or scales is None or (width and width % block != 0):
                raise ValueError("an encoded output needs scales and a block size that divides the width")
            codes = _vector(payload, "payload", device, rows * width, _INT8)
            scale_address = _vector(scales, "scales", device, rows * (width // block) if width else 0, _FLOAT32)
        if inverse_rms is not None:
            inverse = _vector(inverse_rms, "inverse_rms", device, rows, _FLOAT32)
        check("rms_norm_forward", load().nntrain_rms_norm_forward(
            device, kind, x.data_ptr(), x_stride, residual_address, residual_stride, weight_address, _kind(weight), rows,
            width, epsilon, h, y_address, y_kind, codes, scale_address, block_size, inverse,
            _status(finite_status, "finite_status", device), _stream_on(device, stream)))

    @staticmethod
    def backward(device: int, y_gradient, h, weight, inverse_rms, x_gradient, weight_gradient, residual_gradient=None,
                 accumulate: bool = False, workspace=None, stream=None) -> None:
        """From the gradient of y, h = x + residual (what `residual_out` holds, or x)
        and `inverse_rms`: `x_gradient`, the gradient of x and of residual alike,
        plus `residual_gradient`, what reaches h from elsewhere; and
        `weight_gradient` (fp32 or bf16), added to what is there with `accumulate`.
        x_gradient may be y_gradient or residual_gradient itself.  `workspace`
        (optional): uint8 scratch that no call in flight at the same time uses."""
        if h.dim() != 2:
            raise ValueError(f"h has shape {tuple(h.shape)}, expected (rows, width)")
        rows, width = h.shape
        kind = _kind(h)
        same = _BFLOAT16 if kind else _FLOAT32
        h_stride = _rows(h, "h", device, width, same)
        y_stride = _rows(y_gradient, "y_gradient", device, width, same, rows)
        residual_stride = residual_address = 0
        if residual_gradient is not None:
            residual_stride = _rows(residual_gradient, "residual_gradient", device, width, same, rows)
            residual_address = residual_gradient.data_ptr()
        weight_address = _vector(weight, "weight", device, width, _FLOATS)
        inverse = _vector(inverse_rms, "inverse_rms", device, rows, _FLOAT32)
        dx = _vector(x_gradient, "x_gradient", device, rows * width, same)
        dw = _vector(weight_gradient, "weight_gradient", device, width, _FLOATS)
        workspace, bytes_ = _workspace("nntrain_rms_norm_backward_workspace", (rows, width), device, workspace, stream)
        check("rms_norm_backward", load().nntrain_rms_norm_backward(
            device, kind, y_gradient.data_ptr(), y_stride, residual_address, residual_stride, h.data_ptr(), h_stride,
            weight_address, _kind(weight), inverse, rows, width, dx, dw, _kind(weight_gradient), accumulate,
            0 if workspace is None else workspace.data_ptr(), bytes_, _stream_on(device, stream)))


class TokenEmbedding:
    """Rows of a token table times a scale, and the table's gradient.  `tokens` are
    int32 or int64 row numbers, any shape; `padding_token` stands for no token.  A
    token that is neither it nor a row counts as none and sets `token_status`
    (optional, int32) to 1."""

    @staticmethod
    def lookup(device: int, tokens, table, out, scale: float = 1.0, table_scales=None, block_size: int = 0,
               first_value: int = 0, padding_token: int = -1, token_status=None, stream=None) -> None:
        """out[t] = scale * table[tokens[t]], zeros where there is no token.  `table`
        (vocab, width): fp32, bf16 or an int8 payload with the `table_scales` and
        block size of the arena in which it begins at `first_value`.  `out`
        (tokens, width): fp32 or bf16, any row stride."""
        count, bytes_ = _tokens(tokens, device)
        vocab, width, kind = _table(table, "table", device, _FLOATS + _INT8)
        out_stride = _rows(out, "out", device, width, _FLOATS, count)
        scales = 0
        if kind == 2:
            if table_scales is None or block_size < 0 or first_value < 0:
                raise ValueError("an encoded table needs its scales, block size and place in the arena")
            needed = 1 if block_size == 0 else (first_value + vocab * width + block_size - 1) // block_size
            if table_scales.numel() < needed:
                raise ValueError(f"table_scales has {table_scales.numel()} values, needs {needed}")
            scales = _vector(table_scales, "table_scales", device, table_scales.numel(), _FLOAT32)
        elif table_scales is not None:
            raise ValueError("a table that is not encoded has no scales")
        check("embedding_lookup", load().nntrain_embedding_lookup(
            device, kind, table.data_ptr(), scales, block_size, first_value, vocab, width, tokens.data_ptr(), bytes_, count,
            padding_token, scale, _kind(out), out.data_ptr(), out_stride, _status(token_status, "token_status", device),
            _stream_on(device, stream)))

    @staticmethod
    def gradient(device: int, tokens, out_gradient, table_gradient, scale: float = 1.0, accumulate: bool = False,
                 padding_token: int = -1, token_status=None, workspace=None, stream=None) -> None:
        """table_gradient[v] = scale * sum of out_gradient[t] over tokens[t] = v, in
        the order of t: the whole table, or with `accumulate` added to the rows that
        are named.  `out_gradient` (tokens, width) fp32 or bf16, any row stride;
        `table_gradient` (vocab, width) fp32 or bf16, at any place of an arena.
        `workspace` (optional): uint8 scratch that no call in flight at the same
        time uses."""
        count, bytes_ = _tokens(tokens, device)
        vocab, width, kind = _table(table_gradient, "table_gradient", device, _FLOATS)
        stride = _rows(out_gradient, "out_gradient", device, width, _FLOATS, count)
        workspace, workspace_bytes = _workspace("nntrain_embedding_gradient_workspace", (count, vocab, width), device,
                                                workspace, stream)
        check("embedding_gradient", load().nntrain_embedding_gradient(
            device, _kind(out_gradient), out_gradient.data_ptr(), stride, tokens.data_ptr(), bytes_, count, padding_token,
            scale, kind, table_gradient.data_ptr(), vocab, width, accumulate, _status(token_status, "token_status", device),
            0 if workspace is None else workspace.data_ptr(), workspace_bytes, _stream_on(device, stream)))


def _tokens(tokens: torch.Tensor, device: int) -> tuple[int, int]:
    if tokens.dtype not in _INTEGERS:
        raise ValueError(f"tokens must be int32 or int64, got {tokens.dtype}")
    count = tokens.numel()
    _vector(tokens, "tokens", device, count, _INTEGERS)
    return count, 8 if tokens.dtype is torch.int64 else 4


def _table(table: torch.Tensor, name: str, device: int, dtypes) -> tuple[int, int, int]:
    """(rows, width, kind) of a token table."""
    _vector(table, name, device, table.numel(), dtypes)
    shape = table.shape
    if len(shape) != 2 or not shape[0] or not shape[1]:
        raise ValueError(f"{name} has shape {tuple(shape)}, expected (vocab, width)")
    return shape[0], shape[1], 2 if table.dtype is torch.int8 else _kind(table)
