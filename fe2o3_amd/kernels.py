"""Typed kernel launch surface.

Mirrors the reference's generated ``<kernel>_gpu`` modules
(crates/fe2o3-macros/src/lib.rs:1081-1120; the vecadd instance is
crates/fe2o3-host/src/generated_vecadd.rs:37-165):

    k = tiled_gemm_lds_slice1_gpu.Kernel.load(ctx)
    k.prepare(a, b, c).launch(stream)

``load`` checks the device (gfx950 only), ``prepare`` checks every slice's
element type and length against the kernel signature and fails closed with
``Fe2o3Error`` before any launch, and ``launch`` enqueues on the stream and
then synchronizes it, so buffers are quiescent when it returns, as the
reference's typed launch is synchronous by design
(crates/fe2o3-host/src/loaded_kernel.rs:420-432).  The prepared launch holds
its slices, so buffers handed in as temporaries live until it is dropped.
``launch_async`` only enqueues: keep the prepared launch (or the buffers)
until the stream has been synchronized.  The physical argument order is the reference's: one
(pointer, length) pair per slice in declaration order, then the scalars
(examples/tiled_gemm_general_v1/hardware-harness/src/lib.rs:578-597).
"""
from __future__ import annotations

import ctypes as C
import struct

import numpy as np

from . import _lib
from .runtime import DeviceBuffer, Fe2o3Error, GpuContext, Stream, check, stream_handle

U16, U32, F32, U8 = np.dtype(np.uint16), np.dtype(np.uint32), np.dtype(np.float32), np.dtype(np.uint8)
ERR_LENGTH = -2


class _Prepared:
    """A checked launch: the flattened arguments, plus the slices themselves,
    held so that a buffer passed as a temporary (``prepare(ctx.to_device(x),
    ...)``) stays allocated until the launch has run; a DeviceBuffer frees
    its memory when it is collected."""

    def __init__(self, kernel: "_TypedKernel", args: tuple, buffers: tuple):
        self.kernel = kernel
        self.args = args
        self.buffers = buffers

    def launch_async(self, stream: Stream | None = None) -> None:
        fn = getattr(_lib.lib(), self.kernel.ENTRY)
        self.kernel.ctx.bind()
        check(fn(*self.args, stream_handle(stream)), self.kernel.ENTRY)

    def launch(self, stream: Stream | None = None) -> None:
        self.launch_async(stream)
        if stream is None:
            self.kernel.ctx.synchronize()
        else:
            stream.synchronize()


class _TypedKernel:
    ENTRY = ""
    # (name, dtype, fixed length or None) per slice, in declaration order
    SLICES: tuple = ()
    # (name, ctypes type) per scalar, in declaration order
    SCALARS: tuple = ()

    def __init__(self, ctx: GpuContext):
        self.ctx = ctx

    @classmethod
    def load(cls, ctx: GpuContext | None = None):
        return cls(ctx or GpuContext.current())

    def prepare(self, *args) -> _Prepared:
        ns, nk = len(self.SLICES), len(self.SCALARS)
        if len(args) != ns + nk:
            raise TypeError(f"{self.ENTRY} takes {ns} slices and {nk} scalars")
        flat = []
        for (name, dtype, fixed), buf in zip(self.SLICES, args[:ns]):
            if buf is None:
                flat += [None, 0]
                continue
            if not isinstance(buf, DeviceBuffer):
                raise TypeError(f"{name} must be a DeviceBuffer")
            if buf.dtype != dtype:
                raise TypeError(f"{name} must hold {dtype}, not {buf.dtype}")
            if fixed is not None and buf.count != fixed:
                raise Fe2o3Error(ERR_LENGTH, f"{self.ENTRY}: {name} length {buf.count} != {fixed}")
            flat += [buf.ptr, buf.count]
        for (name, ctype), value in zip(self.SCALARS, args[ns:]):
            flat.append(ctype(value))
        return _Prepared(self, tuple(flat), tuple(args[:ns]))


def _typed(entry, slices, scalars=()):
    kernel = type("Kernel", (_TypedKernel,), {"ENTRY": entry, "SLICES": tuple(slices),
                                              "SCALARS": tuple(scalars)})
    return type(entry.replace("fe2o3_", "") + "_gpu", (), {"Kernel": kernel})


u32, i32, f32 = C.c_uint32, C.c_int32, C.c_float

# examples/tiled_gemm_v1/src/kernel.rs:63-67
tiled_gemm_lds_slice1_gpu = _typed(
    "fe2o3_tiled_gemm_lds_slice1_v1", [("a", U16, 256), ("b", U16, 256), ("c", F32, 256)])
# examples/tiled_gemm_v1/src/contract.rs:387-427 (the multi-tile plan)
tiled_gemm_v1_gpu = _typed(
    "fe2o3_tiled_gemm_v1", [("a", U16, None), ("b", U16, None), ("c", F32, None)],
    [("m", u32), ("n", u32), ("k", u32)])
# examples/tiled_gemm_general_v1/src/kernel.rs:67-79
tiled_gemm_general_v1_gpu = _typed(
    "fe2o3_tiled_gemm_general_v1", [("a", U16, None), ("b", U16, None), ("c", F32, None)],
    [("m", u32), ("n", u32), ("k", u32), ("lda", u32), ("ldb", u32), ("ldc", u32),
     ("alpha", f32), ("beta", f32)])
# the same kernel under the VectorizedAOnlyBf16GlobalTransferV1 schedule
# (crates/dialect-schedule/src/general_gemm.rs:13-38)
tiled_gemm_general_vector_a_v1_gpu = _typed(
    "fe2o3_tiled_gemm_general_vector_a_v1",
    [("a", U16, None), ("b", U16, None), ("c", F32, None)],
    [("m", u32), ("n", u32), ("k", u32), ("lda", u32), ("ldb", u32), ("ldc", u32),
     ("alpha", f32), ("beta", f32)])
# examples/scalar_gemm_v1/src/kernel.rs:8
scalar_gemm_v1_gpu = _typed(
    "fe2o3_scalar_gemm_v1", [("a", F32, None), ("b", F32, None), ("c", F32, None)],
    [("m", u32), ("n", u32), ("k", u32)])
# scaled-up bf16 NT GEMM (B stored [n, k])
gemm_bf16_nt_gpu = _typed(
    "fe2o3_gemm_bf16_nt", [("a", U16, None), ("b", U16, None), ("c", U16, None)],
    [("m", u32), ("n", u32), ("k", u32)])
# examples/row_softmax_v1/src/kernel.rs:13
row_softmax_v1_gpu = _typed("fe2o3_row_softmax_v1", [("input", F32, 64), ("output", F32, 64)])
row_softmax_gpu = _typed(
    "fe2o3_row_softmax", [("input", F32, None), ("output", F32, None), ("mask", U8, None)],
    [("rows", C.c_uint64), ("cols", C.c_uint64)])
# examples/flash_attention_v1/src/kernel.rs:130-135
flash_attention_causal_f32_b1_h1_n8_d16_v1_gpu = _typed(
    "fe2o3_flash_attention_causal_f32_b1_h1_n8_d16_v1",
    [("q", F32, 128), ("k", F32, 128), ("v", F32, 128), ("output", F32, 128)])
flash_attention_fwd_gpu = _typed(
    "fe2o3_flash_attention_fwd",
    [("q", U16, None), ("k", U16, None), ("v", U16, None), ("o", U16, None), ("lse", F32, None)],
    [("batch", u32), ("heads", u32), ("seq", u32), ("head_dim", u32), ("causal", i32),
     ("scale", f32)])
# examples/moe_top2_v1/src/kernel.rs:102-111
moe_top2_route_f32_t8_e4_k2_c4_v1_gpu = _typed(
    "fe2o3_moe_top2_route_f32_t8_e4_k2_c4_v1",
    [("logits", F32, 32), ("top2_experts", U32, 16), ("requested_counts", U32, 4),
     ("admitted_counts", U32, 4), ("expert_offsets", U32, 5), ("route_slots", U32, 16),
     ("permutation", U32, 16), ("inverse_permutation", U32, 16)])
# examples/moe_expert_v1/src/kernel.rs:30-34, 104-109
moe_expert_gemm_bf16_m16_n16_k16_v1_gpu = _typed(
    "fe2o3_moe_expert_gemm_bf16_m16_n16_k16_v1",
    [("activations", U16, 256), ("weights", U16, 256), ("output", F32, 256)])
moe_expert_combine_f32_t8_k2_o16_v1_gpu = _typed(
    "fe2o3_moe_expert_combine_f32_t8_k2_o16_v1",
    [("compact_output", F32, 256), ("inverse", U32, 16), ("route_weights", F32, 16),
     ("combined_output", F32, 128)])


# ---- functional helpers for the scaled-up paths -------------------------------------

def _call(entry: str, *args, stream: Stream | None = None, sync: bool = True) -> None:
    fn = getattr(_lib.lib(), entry)
    status = fn(*args, None if stream is None else stream_handle(stream))
    if status != 0:
        check(status, entry)
    if sync:
        if stream is None:
            check(_lib.lib().fe2o3_rt_device_synchronize(), "device synchronize")
        else:
            stream.synchronize()


def _ps(buf: DeviceBuffer | None):
    return (None, 0) if buf is None else (buf.ptr, buf.count)


def moe_top2_route(logits: DeviceBuffer, out: dict, tokens: int, experts: int,
                   capacity: int = 0xFFFFFFFF, stream=None, sync=True) -> None:
    """Top-2 router over bf16 (uint16 buffer) or f32 logits.  ``out`` maps the
    names top2, requested, admitted, offsets, slots, permutation, inverse,
    weights to DeviceBuffers (weights may be absent)."""
    dtype_code = 1 if logits.dtype == U16 else 0
    _call("fe2o3_moe_top2_route", *_ps(logits), dtype_code,
          *_ps(out["top2"]), *_ps(out["requested"]), *_ps(out["admitted"]),
          *_ps(out["offsets"]), *_ps(out["slots"]), *_ps(out["permutation"]),
          *_ps(out["inverse"]), *_ps(out.get("weights")), tokens, experts, capacity,
          stream=stream, sync=sync)


def moe_ffn_workspace_bytes(tokens: int, hidden: int, ffn: int, experts: int) -> int:
    return int(_lib.lib().fe2o3_moe_ffn_workspace_bytes(tokens, hidden, ffn, experts))


def moe_ffn_top2(x, w_gate, w_up, w_down, routing: dict, out, workspace, tokens, hidden, ffn,
                 experts, stream=None, sync=True) -> None:
    _call("fe2o3_moe_ffn_top2", *_ps(x), *_ps(w_gate), *_ps(w_up), *_ps(w_down),
          *_ps(routing["top2"]), *_ps(routing["offsets"]), *_ps(routing["permutation"]),
          *_ps(routing["inverse"]), *_ps(routing["weights"]), *_ps(out),
          workspace.ptr, workspace.nbytes, tokens, hidden, ffn, experts,
          stream=stream, sync=sync)


def moe_ffn_top2_noalloc(x, w_gate, w_up, w_down, routing: dict, out, tokens, hidden, ffn,
                         experts, stream=None, sync=True) -> None:
    """fe2o3_moe_ffn_top2 without a workspace argument: the library's own
    per-device scratch (FE2O3_MOE_NOALLOC_SCRATCH_BYTES), no allocation."""
    _call("fe2o3_moe_ffn_top2_noalloc", *_ps(x), *_ps(w_gate), *_ps(w_up), *_ps(w_down),
          *_ps(routing["top2"]), *_ps(routing["offsets"]), *_ps(routing["permutation"]),
          *_ps(routing["inverse"]), *_ps(routing["weights"]), *_ps(out), tokens, hidden, ffn,
          experts, stream=stream, sync=sync)


def amax_f32(x: DeviceBuffer, amax: DeviceBuffer, stream=None, sync=True) -> None:
    _call("fe2o3_amax_f32", x.ptr, x.count, amax.ptr, stream=stream, sync=sync)


def fp8_scale_from_amax(amax: DeviceBuffer, scale: DeviceBuffer, stream=None, sync=True) -> None:
    _call("fe2o3_fp8_scale_from_amax", amax.ptr, scale.ptr, stream=stream, sync=sync)


def quantize_e4m3(x: DeviceBuffer, scale: DeviceBuffer, q: DeviceBuffer, stream=None,
                  sync=True) -> None:
    _call("fe2o3_quantize_e4m3", x.ptr, x.count, scale.ptr, q.ptr, q.count, stream=stream,
          sync=sync)


# gfx942 FNUZ fp8 formats (FE2O3_FP8_FNUZ_E4M3 / _E5M2)
FNUZ_E4M3, FNUZ_E5M2 = 0, 1


def fp8_fnuz_from_f32(x: DeviceBuffer, q: DeviceBuffer, fmt: int, stream=None,
                      sync=True) -> None:
    """q = Fp8E4M3Fnuz / Fp8E5M2Fnuz::from_f32(x) elementwise
    (crates/fe2o3-device/src/fp8.rs:85-95, 193-203)."""
    _call("fe2o3_fp8_fnuz_from_f32", x.ptr, x.count, q.ptr, q.count, fmt, stream=stream,
          sync=sync)


def fp8_fnuz_to_f32(q: DeviceBuffer, x: DeviceBuffer, fmt: int, stream=None,
                    sync=True) -> None:
    """x = Fp8E4M3Fnuz / Fp8E5M2Fnuz::to_f32(q) elementwise
    (crates/fe2o3-device/src/fp8.rs:92-95, 200-203)."""
    _call("fe2o3_fp8_fnuz_to_f32", q.ptr, q.count, x.ptr, x.count, fmt, stream=stream,
          sync=sync)


def bf16_from_f32(x: DeviceBuffer, out: DeviceBuffer, stream=None, sync=True) -> None:
    """out = Bf16::from_f32(x) elementwise (crates/fe2o3-device/src/half.rs:182-190)."""
    _call("fe2o3_bf16_from_f32", x.ptr, x.count, out.ptr, out.count, stream=stream, sync=sync)


def gemm_fp8_nt(a, b, scale_a, scale_b, c, m, n, k, stream=None, sync=True) -> None:
    _call("fe2o3_gemm_fp8_nt", a.ptr, a.count, b.ptr, b.count, scale_a.ptr, scale_b.ptr,
          c.ptr, c.count, m, n, k, stream=stream, sync=sync)


# examples/wave64_collectives_v1/src/kernel.rs:18-67 (the mask is a scalar
# between the input slice and the three output slices)
def wave64_collectives_v1(input: DeviceBuffer, active_mask: int, reduction: DeviceBuffer,
                          inclusive: DeviceBuffer, exclusive: DeviceBuffer, stream=None,
                          sync=True) -> None:
    _call("fe2o3_wave64_collectives_v1", *_ps(input), C.c_uint64(active_mask & (2**64 - 1)),
          *_ps(reduction), *_ps(inclusive), *_ps(exclusive), stream=stream, sync=sync)


def wave64_collectives_rows(input: DeviceBuffer, masks: DeviceBuffer, reduction: DeviceBuffer,
                            inclusive: DeviceBuffer, exclusive: DeviceBuffer, rows: int,
                            stream=None, sync=True) -> None:
    _call("fe2o3_wave64_collectives_rows", *_ps(input), *_ps(masks), *_ps(reduction),
          *_ps(inclusive), *_ps(exclusive), rows, stream=stream, sync=sync)


# examples/workgroup_sync_v1/src/kernel.rs:18-78
def lds_reduce_i32_v1(values: DeviceBuffer, output: DeviceBuffer, stream=None,
                      sync=True) -> None:
    _call("fe2o3_lds_reduce_i32_v1", *_ps(values), *_ps(output), stream=stream, sync=sync)


# examples/workgroup_sync_v1/src/scoped_atomic.rs:11-32 (target: one u32)
def scoped_atomic_add_u32_v1(values: DeviceBuffer, eligible: DeviceBuffer,
                             target: DeviceBuffer, stream=None, sync=True) -> None:
    _call("fe2o3_scoped_atomic_add_u32_v1", *_ps(values), *_ps(eligible), target.ptr,
          stream=stream, sync=sync)


# crates/fe2o3-host/src/moe_routing_expert_bridge_v1.rs:220-389 on the device;
# record: 4 x u32 {kind, index, expected, actual}
def moe_routing_check(routing: dict, tokens: int, experts: int, capacity: int,
                      record: DeviceBuffer, stream=None, sync=True) -> None:
    _call("fe2o3_moe_routing_check", *_ps(routing["top2"]), *_ps(routing["requested"]),
          *_ps(routing["admitted"]), *_ps(routing["offsets"]), *_ps(routing["slots"]),
          *_ps(routing["permutation"]), *_ps(routing["inverse"]), tokens, experts, capacity,
          *_ps(record), stream=stream, sync=sync)


# ---- paged key-value cache ---------------------------------------------------------------
#
# Calls go to `stream`, the null stream if None, whatever stream is torch's current
# one: order them behind what writes their tensors, and without sync keep the
# tensors until the stream is through.

KV_BF16, KV_E4M3, KV_MXFP4 = 0, 1, 4
KV_NO_SLOT = 0xFFFFFFFF
MXFP4_BLOCK, MXFP4_PANEL = 32, 256
PAGED_ATTENTION_MAX_WORKGROUPS = 768

# what an array of each kind may hold: element types of a DeviceBuffer, and of
# a tensor
_BF16, _CODES, _INDEX, _FLOAT, _BYTES, _DOUBLE = (
    "bf16", "e4m3", "u32", "f32", "bytes", "f64")
_HOLDS = {
    _BF16: ("uint16", "torch.bfloat16"),
    _CODES: ("uint8", "torch.uint8", "torch.float8_e4m3fn"),
    _INDEX: ("uint32", "torch.int32", "torch.uint32"),
    _FLOAT: ("float32", "torch.float32"),
    _BYTES: ("uint8", "torch.uint8", "torch.int8"),
    _DOUBLE: ("float64", "torch.float64"),
}


class _Kinds(dict):
    """element type -> the kinds it may stand for"""

    def __missing__(self, dtype):
        found = self[dtype] = frozenset(k for k, v in _HOLDS.items() if str(dtype) in v)
        return found


_kinds = _Kinds()


class _Is(dict):
    """element type -> whether it may stand for one kind"""

    def __init__(self, kind):
        super().__init__()
        self.kind = kind

    def __missing__(self, dtype):
        found = self[dtype] = self.kind in _kinds[dtype]
        return found


_is_bf16, _is_codes, _is_index, _is_float, _is_bytes, _is_double = (
    _Is(kind) for kind in (_BF16, _CODES, _INDEX, _FLOAT, _BYTES, _DOUBLE))

# A call of small arrays takes longer here than on the device, so calls with tensors that
# are all as they should be go by short ways (the _fast functions), which look at each
# thing once; these give None, or fail, for everything else (broadcast or wrong operands),
# and the long way takes it or says what is wrong.  DeviceBuffers go the long way at once: an
# exception takes 0.5 us.
_NOT_FAST = (AttributeError, TypeError, ValueError, KeyError, IndexError, struct.error)


def _at(x, is_kind, device):
    """Address of a contiguous tensor of this kind on the device; None of another."""
    if is_kind[x.dtype] and x.get_device() == device and x.is_contiguous():
        return x.data_ptr()
    return None


def _fast_count(x, shape, strides):
    """Elements that a tensor's strides span."""
    return x.numel() if x.is_contiguous() else _extent(shape, strides, "")


def _operand(x, kind, name, device, dense=True):
    """(pointer, elements) of a DeviceBuffer or a tensor that holds `kind` on
    `device`.  dense: the tensor is contiguous; otherwise its last dimension
    is, and the elements are the extent that its strides span."""
    if isinstance(x, DeviceBuffer):
        if kind not in _kinds[x.dtype]:
            raise TypeError(f"{name} must hold {kind}, not {x.dtype}")
        if x.ctx.device != device:
            raise ValueError(f"{name} on device {x.ctx.device}, not {device}")
        return x.ptr, x.count
    if not hasattr(x, "data_ptr"):
        raise TypeError(f"{name} must be a DeviceBuffer or a device tensor")
    if kind not in _kinds[x.dtype]:
        raise TypeError(f"{name} must hold {kind}, not {x.dtype}")
    where = x.get_device()
    if where != device:
        if where < 0:
            raise TypeError(f"{name} must be in device memory")
        raise ValueError(f"{name} on device {where}, not {device}")
    if x.is_contiguous():
        return x.data_ptr(), x.numel()
    if dense:
        raise ValueError(f"{name} must be contiguous")
    return x.data_ptr(), _extent(x.shape, x.stride(), name)


def _extent(shape, strides, name):
    """Elements that a tensor's strides span; its last dimension is contiguous."""
    if 0 in shape:
        return 0
    if strides[-1] != 1 and shape[-1] != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    count = 1
    for n, stride in zip(shape, strides):
        count += (n - 1) * stride
    return count


def _table(block_table, seqs, device):
    """(pointer, elements, columns) of a block table, flat or [seqs, columns].  A flat
    one of no sequences may have any number of columns: the most."""
    ptr, count = _operand(block_table, _INDEX, "block_table", device)
    shape = getattr(block_table, "shape", None)
    if shape is not None and len(shape) != 1 and shape[0] != seqs:
        raise ValueError(f"a block table of {tuple(shape)} for {seqs} sequences")
    if seqs == 0:
        return ptr, count, shape[1] if shape is not None and len(shape) == 2 else 0xFFFFFFFF
    return ptr, count, count // seqs


def _dimensions(x, dims, name):
    """Shape of a tensor of `dims` dimensions; None of a DeviceBuffer."""
    if isinstance(x, DeviceBuffer):
        return None
    shape = getattr(x, "shape", None)
    if shape is None or len(shape) != dims:
        raise ValueError(f"{name} must be a DeviceBuffer or a tensor of {dims} dimensions")
    return shape


def _same_strides(x, y):
    """Whether two tensors of one shape have the same strides, but for dimensions of
    one, whose stride says nothing."""
    return all(n == 1 or s == t for n, s, t in zip(x.shape, x.stride(), y.stride()))


def _pair(k, v, dims, kind, device):
    """Shape and strides of K and V (None of DeviceBuffers), which are the same for
    both, and (pointer, elements) of each."""
    shape = _dimensions(k, dims, "k")
    if shape is None or isinstance(v, DeviceBuffer):
        return None, None, _operand(k, kind, "k", device) + _operand(v, kind, "v", device)
    strides = k.stride()
    if v.shape != shape or (v.stride() != strides and not _same_strides(k, v)):
        raise ValueError("k and v must have the same shape and strides")
    if (k.get_device() != device or v.get_device() != device or kind not in _kinds[k.dtype]
            or kind not in _kinds[v.dtype]):  # which says what is wrong
        _operand(k, kind, "k", device, False)
        _operand(v, kind, "v", device, False)
    count = k.numel() if k.is_contiguous() else _extent(shape, strides, "k and v")
    return shape, strides, (k.data_ptr(), count, v.data_ptr(), count)


_KV_RECORD = struct.Struct("=11Q6I")  # Fe2o3KvCacheV1


class KvCache:
    """A paged key-value cache: K and V rows in slots page * page_size + place: bf16;
    e4m3 codes with f32 scales [pages, kv_heads, page_size]; or microscaled 4-bit
    codes, two to a byte, with scale bytes [pages, kv_heads, page_size, head_dim / 32].

    k and v are device tensors [pages, page_size, kv_heads, head_dim] (4-bit:
    head_dim / 2 bytes) of any strides but the last (a cache laid out [pages,
    kv_heads, page_size, head_dim] is passed as its transpose(1, 2)), or
    DeviceBuffers with `shape` given that way and `strides` (page, token, head;
    dense by default) in elements (4-bit: the shape with head_dim, the strides in
    bytes).  K and V have the same strides; scales of bytes make the cache a 4-bit
    one.  The record holds the arrays, not copies of them.
    """

    def __init__(self, k, v, k_scale=None, v_scale=None, *, shape=None, strides=None):
        try:
            record = self._fast(k, v, k_scale, v_scale) if shape is None else None
        except _NOT_FAST:
            record = None
        if record is not None:
            self.arrays = (k, v, k_scale, v_scale)
            self.record = _lib.Fe2o3KvCacheV1.from_buffer_copy(record)
            return
        if (k_scale is None) != (v_scale is None):
            raise ValueError("k_scale and v_scale go together")
        self.device = device = _device_of(k)
        packed = 1  # elements in one of the array's
        if k_scale is None:
            self.format, kind = KV_BF16, _BF16
        elif _BYTES in _kinds[k_scale.dtype]:
            self.format, kind, packed = KV_MXFP4, _BYTES, 2
        else:
            self.format, kind = KV_E4M3, _CODES
        found, found_strides, arrays = _pair(k, v, 4, kind, device)
        if found is not None:
            pages, page_size, kv_heads, width = found
            strides, head_dim = found_strides[:3], packed * width
        elif shape is None:
            raise ValueError("a cache of DeviceBuffers needs its shape")
        else:
            pages, page_size, kv_heads, head_dim = shape
        self.shape = (pages, page_size, kv_heads, head_dim)
        if strides is None:
            row = head_dim // packed
            strides = (page_size * kv_heads * row, kv_heads * row, row)
        self.arrays = (k, v, k_scale, v_scale)
        scales = (None, 0, None, 0)
        if k_scale is not None:
            want, scale_kind = (pages, kv_heads, page_size), _FLOAT
            if packed == 2:
                want, scale_kind = want + (head_dim // MXFP4_BLOCK,), _BYTES
            for scale in (k_scale, v_scale):
                found = _dimensions(scale, len(want), "scales")
                if found is not None and found != want:
                    raise ValueError(f"scales of {tuple(found)}, not {want}")
            scales = (_operand(k_scale, scale_kind, "k_scale", device)
                      + _operand(v_scale, scale_kind, "v_scale", device))
        self.record = _lib.Fe2o3KvCacheV1(*arrays, *scales, *strides, self.format, pages, page_size,
                                          kv_heads, head_dim, 0)

    def _fast(self, k, v, k_scale, v_scale):
        shape, found, device = k.shape, k.stride(), k.get_device()
        if (device < 0 or v.get_device() != device or v.shape != shape or v.stride() != found
                or (found[3] != 1 and shape[3] != 1)):
            return None
        pages, page_size, kv_heads, head_dim = shape
        count = _fast_count(k, shape, found)
        ks = vs = scales = 0
        if k_scale is None:
            fmt, is_kind = KV_BF16, _is_bf16
            if v_scale is not None:
                return None
        else:
            want = (pages, kv_heads, page_size)
            if _is_bytes[k_scale.dtype]:
                fmt, is_kind, is_scale = KV_MXFP4, _is_bytes, _is_bytes
                head_dim *= 2
                want += (head_dim // MXFP4_BLOCK,)
            else:
                fmt, is_kind, is_scale = KV_E4M3, _is_codes, _is_float
            ks, vs = _at(k_scale, is_scale, device), _at(v_scale, is_scale, device)
            if ks is None or vs is None or k_scale.shape != want or v_scale.shape != want:
                return None
            scales = k_scale.numel()
        if not (is_kind[k.dtype] and is_kind[v.dtype]):
            return None
        record = _KV_RECORD.pack(k.data_ptr(), count, v.data_ptr(), count, ks, scales, vs, scales,
                                 *found[:3], fmt, pages, page_size, kv_heads, head_dim, 0)
        self.device, self.format = device, fmt
        self.shape = (pages, page_size, kv_heads, head_dim)
        return record


def _device_of(k):
    if isinstance(k, DeviceBuffer):
        return k.ctx.device
    if not hasattr(k, "get_device"):
        raise TypeError("k must be a DeviceBuffer or a device tensor")
    device = k.get_device()
    if device < 0:
        raise TypeError("a cache lies in device memory")
    return device


def _on_current_device(cache):
    """The cache's device, which has to be the current one: launches go there."""
    current = _current_device()
    if current != cache.device:
        raise ValueError(f"cache on device {cache.device}, the current one is {current}")
    return cache.device


def _current_device():
    current = C.c_int32()
    status = _lib.lib().fe2o3_rt_get_device(C.byref(current))
    if status != 0:
        check(status, "get device")
    return current.value


def _rows(cache, k, v, strides, device):
    """K and V rows of a cache's heads: tokens (None of DeviceBuffers), (token, head)
    strides, and (pointer, elements) of each."""
    _, _, kv_heads, head_dim = cache.shape
    shape, found, arrays = _pair(k, v, 3, _BF16, device)
    if shape is None:
        return None, strides or (kv_heads * head_dim, head_dim), arrays
    if shape[1] != kv_heads or shape[2] != head_dim:
        raise ValueError(f"rows of {tuple(shape[1:])} for a cache of {(kv_heads, head_dim)}")
    return shape[0], found[:2], arrays


def _fast_rows(cache, k, v, device):
    """(tokens, token stride, head stride, address and elements of K and of V) of rows in
    tensors."""
    shape, strides = k.shape, k.stride()
    tokens, kv_heads, head_dim = shape
    if (kv_heads != cache.shape[2] or head_dim != cache.shape[3] or v.shape != shape
            or v.stride() != strides or (strides[2] != 1 and head_dim != 1)
            or k.get_device() != device or v.get_device() != device
            or not (_is_bf16[k.dtype] and _is_bf16[v.dtype])):
        return None
    count = _fast_count(k, shape, strides)
    return tokens, strides[0], strides[1], k.data_ptr(), count, v.data_ptr(), count


def kv_cache_write(cache: KvCache, k, v, slots, *, strides=None, stream=None, sync=True) -> None:
    """Writes rows k, v (bf16 [tokens, kv_heads, head_dim]; DeviceBuffers with
    `strides` (token, head)) into slots[t] of the cache, quantised where it is
    e4m3 or 4-bit.  A slot out of range (KV_NO_SLOT) is skipped; each slot at most once
    a call (fe2o3_kv_cache_write)."""
    device = _on_current_device(cache)
    rows = None
    if strides is None and not isinstance(k, DeviceBuffer):
        try:
            rows = _fast_rows(cache, k, v, device)
            slots_ptr = _at(slots, _is_index, device)
        except _NOT_FAST:
            rows = None
    if rows is not None and slots_ptr is not None and slots.numel() == rows[0]:
        tokens = rows[0]
        _call("fe2o3_kv_cache_write", C.byref(cache.record), *rows[3:], slots_ptr, tokens, tokens,
              rows[1], rows[2], stream=stream, sync=sync)
        return
    rows, strides, arrays = _rows(cache, k, v, strides, device)
    slots_ptr, tokens = _operand(slots, _INDEX, "slots", device)
    if rows is not None and rows != tokens:
        raise ValueError(f"{rows} rows and {tokens} slots")
    _call("fe2o3_kv_cache_write", C.byref(cache.record), *arrays, slots_ptr, tokens, tokens,
          *strides, stream=stream, sync=sync)


def kv_cache_read(cache: KvCache, block_table, starts, k, v, *, strides=None, tokens=None,
                  stream=None, sync=True) -> None:
    """Reads cached rows into k, v (bf16 [tokens, kv_heads, head_dim]): sequence
    s, on pages block_table[s], to rows starts[s] .. starts[s + 1] - 1.  Rows in
    no sequence keep their values (fe2o3_kv_cache_read).  DeviceBuffers take
    `strides` (token, head) and `tokens`."""
    device = _on_current_device(cache)
    rows = None
    if strides is None and tokens is None:
        try:
            rows = _fast_rows(cache, k, v, device)
            table_ptr = _at(block_table, _is_index, device)
            starts_ptr = _at(starts, _is_index, device)
            (seqs, cols), starts_len = block_table.shape, starts.numel()
        except _NOT_FAST:
            rows = None
    if (rows is not None and table_ptr is not None and starts_ptr is not None
            and starts_len == seqs + 1):
        _call("fe2o3_kv_cache_read", C.byref(cache.record), table_ptr, seqs * cols, starts_ptr,
              starts_len, *rows[3:], seqs, cols, rows[0], rows[1], rows[2], stream=stream,
              sync=sync)
        return
    rows, strides, arrays = _rows(cache, k, v, strides, device)
    starts_ptr, starts_len = _operand(starts, _INDEX, "starts", device)
    seqs = starts_len - 1
    if seqs < 0:
        raise ValueError("starts must hold one value more than there are sequences")
    table_ptr, table_len, cols = _table(block_table, seqs, device)
    if rows is None:
        rows = arrays[1] // (cache.shape[2] * cache.shape[3]) if tokens is None else tokens
    _call("fe2o3_kv_cache_read", C.byref(cache.record), table_ptr, table_len, starts_ptr,
          starts_len, *arrays, seqs, cols, rows, *strides, stream=stream, sync=sync)


def paged_attention_workspace_bytes(q_heads: int, kv_heads: int, head_dim: int) -> int:
    """FE2O3_PAGED_ATTENTION_WORKSPACE_BYTES: scratch of one decode call."""
    rows = min(q_heads // kv_heads, 64)
    if kv_heads % 4 == 0 and rows <= 16:  # four heads at once
        rows *= 4
    return PAGED_ATTENTION_MAX_WORKGROUPS * 8 * (head_dim + 2) * rows


def _fast_decode(cache, q, block_table, lengths, out, lse, workspace, device):
    """The call's arguments but max_length, window and scale, of tensors; None if they are
    not as they should be."""
    shape, strides = q.shape, q.stride()
    seqs, q_heads, head_dim = shape
    found_seqs, cols = block_table.shape
    heads = seqs * q_heads
    table_at, lengths_at = _at(block_table, _is_index, device), _at(lengths, _is_index, device)
    out_at, work_at = _at(out, _is_bf16, device), _at(workspace, _is_bytes, device)
    lse_at = 0 if lse is None else _at(lse, _is_float, device)
    if (None in (table_at, lengths_at, out_at, work_at, lse_at) or not seqs
            or found_seqs != seqs or lengths.numel() != seqs or head_dim != cache.shape[3]
            or (strides[1] != head_dim and q_heads != 1) or (strides[2] != 1 and head_dim != 1)
            or not _is_bf16[q.dtype] or q.get_device() != device or out.shape != shape
            or (lse is not None and lse.shape != (seqs, q_heads))):
        return None
    return (q.data_ptr(), _fast_count(q, shape, strides), table_at, seqs * cols, lengths_at, seqs,
            out_at, heads * head_dim, lse_at, 0 if lse is None else heads, work_at,
            workspace.numel(), seqs, q_heads, cols, strides[0])


def paged_attention_decode(cache: KvCache, q, block_table, lengths, out, lse, workspace, *,
                           max_length: int, scale: float, window: int = 0, q_heads=None,
                           q_stride=None, stream=None, sync=True) -> None:
    """Attention of one new token per sequence over its cached keys: q and out
    bf16 [seqs, q_heads, head_dim], lse f32 [seqs, q_heads] or None, block_table
    [seqs, cols], lengths [seqs], at most max_length each; window > 0 keeps the
    last `window` keys (fe2o3_paged_attention_decode).  workspace: device bytes,
    paged_attention_workspace_bytes at least, of no use to another call that may
    overlap.  out and lse may be flat.  DeviceBuffers take q_heads, and q_stride
    between sequences."""
    device = _on_current_device(cache)
    try:
        args = (_fast_decode(cache, q, block_table, lengths, out, lse, workspace, device)
                if q_heads is None and q_stride is None else None)
    except _NOT_FAST:
        args = None
    if args is not None:
        _call("fe2o3_paged_attention_decode", C.byref(cache.record), *args[:-4], *args[-4:-1],
              max_length, args[-1], window, scale, stream=stream, sync=sync)
        return
    head_dim = cache.shape[3]
    lengths_ptr, seqs = _operand(lengths, _INDEX, "lengths", device)
    shape = _dimensions(q, 3, "q")
    if shape is not None:
        rows, q_heads, width = shape
        q_stride, head_stride, _ = q.stride()
        if rows != seqs:
            raise ValueError(f"{rows} rows of q and {seqs} lengths")
        if width != head_dim or (head_stride != width and q_heads != 1):
            raise ValueError("q must be [seqs, q_heads, head_dim] with a sequence's heads dense")
    elif q_heads is None:
        raise ValueError("q in a DeviceBuffer needs q_heads")
    elif q_stride is None:
        q_stride = q_heads * head_dim
    for name, x, want in (("out", out, (seqs, q_heads, head_dim)), ("lse", lse, (seqs, q_heads))):
        found = getattr(x, "shape", want)
        if found != want and len(found) != 1:
            raise ValueError(f"{name} of {tuple(found)}, not {want}")
    table_ptr, table_len, cols = _table(block_table, seqs, device)
    lse_ptr, lse_len = (None, 0) if lse is None else _operand(lse, _FLOAT, "lse", device)
    _call("fe2o3_paged_attention_decode", C.byref(cache.record),
          *_operand(q, _BF16, "q", device, False), table_ptr, table_len, lengths_ptr, seqs,
          *_operand(out, _BF16, "out", device), lse_ptr, lse_len,
          *_operand(workspace, _BYTES, "workspace", device), seqs, q_heads, cols, max_length,
          q_stride, window, scale, stream=stream, sync=sync)


# ---- rotary positions ----------------------------------------------------------------------

ROTARY_INTERLEAVED, ROTARY_INVERSE = 1, 2


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, factor: float = 1.0,
                       schedule: str = "linear", original_length: int = 4096,
                       slow_turns: float = 1.0, fast_turns: float = 32.0):
    """(radians a position for each pair, in 64 bits, numpy; the scale of rotary()) for a
    context `factor` times as long as the model's own original_length:

      "linear"    every pair factor times slower
      "base"      base stretched, so that the slowest pair is factor times slower and the
                  fastest keeps its speed
      "by_turns"  pairs of fast_turns and more over original_length keep their speed,
                  those of slow_turns and fewer are factor times slower, a straight line
                  in the turns between, as Peng, Quesnelle, Fan and Shippole publish it
                  (YaRN, 2023); the scale is 0.1 ln(factor) + 1.  A model whose program
                  draws that line over the pairs' numbers has other angles: make their
                  table as it does, rotary() takes any
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be positive and even")
    if base <= 0 or factor <= 0 or original_length <= 0 or not 0 <= slow_turns < fast_turns:
        raise ValueError("base, factor and original_length must be positive, "
                         "and slow_turns below fast_turns")
    if schedule not in ("linear", "base", "by_turns"):
        raise ValueError(f"no schedule {schedule!r}")
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    if schedule == "base":
        if rotary_dim > 2:
            base = base * factor ** (rotary_dim / (rotary_dim - 2))
        return base ** (-2.0 * i / rotary_dim), 1.0
    freq = base ** (-2.0 * i / rotary_dim)
    if schedule == "linear":
        return freq / factor, 1.0
    turns = original_length * freq / (2.0 * np.pi)
    keep = np.clip((turns - slow_turns) / (fast_turns - slow_turns), 0.0, 1.0)
    return freq * (keep + (1.0 - keep) / factor), 0.1 * float(np.log(max(factor, 1.0))) + 1.0


def _rotary_rows(x, out, name, kind, device, tokens, shape, strides):
    """The record of an array's rows, (tokens, heads, head_dim)."""
    found = _dimensions(x, 3, name)
    if found is None:
        if shape is None:
            raise ValueError(f"{name} in a DeviceBuffer needs its heads and head_dim")
        found = (tokens, *shape)
        given = strides or (shape[0] * shape[1], shape[1])
    else:
        given = x.stride()[:2]
    if out is None or out is x:
        out, out_strides = x, given
    else:
        out_shape = _dimensions(out, 3, name + "_out")
        if out_shape is not None and tuple(out_shape) != tuple(found):
            raise ValueError(f"{name}_out of {tuple(out_shape)}, not {tuple(found)}")
        out_strides = (out.stride()[:2] if out_shape is not None
                       else (found[1] * found[2], found[2]))
    ptr, count = _operand(x, kind, name, device, False)
    out_ptr, out_count = (ptr, count) if out is x else _operand(out, kind, name + "_out", device,
                                                                False)
    return _lib.Fe2o3RotaryRowsV1(ptr, count, out_ptr, out_count, *given, *out_strides, found[1],
                                  0), found


_ROTARY_RECORD = struct.Struct("=8Q2I")  # Fe2o3RotaryRowsV1


def _fast_rotary_rows(x, out, is_kind, device):
    """The packed record of rows in tensors, and their shape."""
    shape, given = x.shape, x.stride()
    if not is_kind[x.dtype] or x.get_device() != device or (given[2] != 1 and shape[2] != 1):
        return None
    ptr, count = x.data_ptr(), _fast_count(x, shape, given)
    if out is None:
        out_ptr, out_count, out_strides = ptr, count, given
    else:
        out_strides = out.stride()
        if (out.shape != shape or not is_kind[out.dtype] or out.get_device() != device
                or (out_strides[2] != 1 and shape[2] != 1)):
            return None
        out_ptr, out_count = out.data_ptr(), _fast_count(out, shape, out_strides)
    return _ROTARY_RECORD.pack(ptr, count, out_ptr, out_count, given[0], given[1], out_strides[0],
                               out_strides[1], shape[1], 0), shape


def _fast_rotary(q, k, positions, freq, q_out, k_out, device):
    """The call's arguments before its flags, of tensors."""
    is_float = _is_float[q.dtype]
    is_kind = _is_float if is_float else _is_bf16
    found = _fast_rotary_rows(q, q_out, is_kind, device)
    other = None if k is None else _fast_rotary_rows(k, k_out, is_kind, device)
    positions_at, freq_at = _at(positions, _is_index, device), _at(freq, _is_double, device)
    if found is None or (other is None) != (k is None) or positions_at is None or freq_at is None:
        return None
    record, (tokens, _, head_dim) = found
    pairs = freq.numel()
    if positions.numel() != tokens:
        return None
    if other is not None:
        other, shape = other
        if shape[0] != tokens or shape[2] != head_dim:
            return None
    return (record, other, positions_at, tokens, freq_at, pairs, 0 if is_float else 1, tokens,
            head_dim, 2 * pairs)


def rotary(q, k, positions, freq, *, q_out=None, k_out=None, interleaved=False, inverse=False,
           scale=1.0, q_shape=None, k_shape=None, q_strides=None, k_strides=None, stream=None,
           sync=True) -> None:
    """Turns the first 2 len(freq) elements of every head of q and k, f32 or bf16 [tokens,
    heads, head_dim] (k may be None), by positions [tokens] times freq (f64 radians a
    position, device memory), in place or into q_out and k_out (fe2o3_rotary).
    inverse turns back, for gradients.  DeviceBuffers take their (heads, head_dim) as
    q_shape and k_shape and (token, head) strides, dense by default; outputs in
    DeviceBuffers are dense."""
    device = _current_device()
    flags = ROTARY_INTERLEAVED * bool(interleaved) + ROTARY_INVERSE * bool(inverse)
    try:
        args = (None if isinstance(q, DeviceBuffer)
                else _fast_rotary(q, k, positions, freq, q_out, k_out, device))
    except _NOT_FAST:
        args = None
    if args is not None:
        _call("fe2o3_rotary", *args, flags, scale, stream=stream, sync=sync)
        return
    positions_ptr, tokens = _operand(positions, _INDEX, "positions", device)
    freq_ptr, pairs = _operand(freq, _DOUBLE, "freq", device)
    kind = _FLOAT if _FLOAT in _kinds[q.dtype] else _BF16
    record, shape = _rotary_rows(q, q_out, "q", kind, device, tokens, q_shape, q_strides)
    rows, other = (shape[0],), None
    if k is not None:
        other, k_found = _rotary_rows(k, k_out, "k", kind, device, tokens, k_shape, k_strides)
        if k_found[2] != shape[2]:
            raise ValueError(f"head_dim of {shape[2]} in q and {k_found[2]} in k")
        rows += (k_found[0],)
        other = C.byref(other)
    if any(n != tokens for n in rows):
        raise ValueError(f"{rows} rows and {tokens} positions")
    _call("fe2o3_rotary", C.byref(record), other, positions_ptr, tokens, freq_ptr, pairs,
          kind == _BF16, tokens, shape[2], 2 * pairs, flags, scale, stream=stream, sync=sync)


# ---- microscaled 4-bit matrices ----------------------------------------------------------
#
# Arrays are DeviceBuffers or device tensors, on the current device; streams as for the
# paged cache.


def mxfp4_shapes(rows: int, cols: int) -> tuple[tuple, tuple]:
    """Shapes of a packed matrix's codes and scales, both bytes."""
    panels = -(-cols // MXFP4_PANEL)
    return (rows, panels * 128), (panels, -(-rows // 16) * 16, 8)


def _packed(codes, scales, names, device):
    """(pointer, bytes) of codes and of scales, and their shapes where they are tensors."""
    shapes = _dimensions(codes, 2, names[0]), _dimensions(scales, 3, names[1])
    return (_operand(codes, _BYTES, names[0], device)
            + _operand(scales, _BYTES, names[1], device)), shapes


def _dense(x, name, device, rows, cols, stride):
    """(pointer, elements, dtype code, rows, columns, row stride) of a matrix of f32 or
    bf16: a tensor's own, a DeviceBuffer's as given."""
    kind = _FLOAT if _FLOAT in _kinds[x.dtype] else _BF16
    shape = _dimensions(x, 2, name)
    if shape is not None:
        if (rows, cols, stride) != (None, None, None):
            raise ValueError(f"{name} has its own rows, cols and stride")
        rows, cols = shape
        stride = x.stride()[0]
    elif rows is None or cols is None:
        raise ValueError(f"{name} in a DeviceBuffer needs rows and cols")
    elif stride is None:
        stride = cols
    return _operand(x, kind, name, device, False) + (kind == _BF16, rows, cols, stride)


def _fast_packing(x, codes, scales, device):
    """x, its elements and dtype code, the packed arrays, rows, cols and stride, of tensors."""
    shape, strides = x.shape, x.stride()
    rows, cols = shape
    is_float = _is_float[x.dtype]
    codes_at, scales_at = _at(codes, _is_bytes, device), _at(scales, _is_bytes, device)
    panels = (cols + 255) // 256
    scale_rows = (rows + 15) // 16 * 16
    if (codes_at is None or scales_at is None or codes.shape != (rows, panels * 128)
            or scales.shape != (panels, scale_rows, 8) or not (is_float or _is_bf16[x.dtype])
            or x.get_device() != device or (strides[1] != 1 and cols != 1)):
        return None
    return (x.data_ptr(), _fast_count(x, shape, strides), 0 if is_float else 1, codes_at,
            rows * panels * 128, scales_at, panels * scale_rows * 8, rows, cols, strides[0])


def quantize_mxfp4(x, codes, scales, *, rows=None, cols=None, stride=None, stream=None,
                   sync=True) -> None:
    """Packs x, f32 or bf16 [rows, cols] with the last dimension contiguous, into codes and
    scales of mxfp4_shapes(rows, cols) (fe2o3_quantize_mxfp4).  A DeviceBuffer x takes
    rows, cols and the elements between rows."""
    device = _current_device()
    try:
        args = (_fast_packing(x, codes, scales, device)
                if rows is None and cols is None and stride is None else None)
    except _NOT_FAST:
        args = None
    if args is not None:
        _call("fe2o3_quantize_mxfp4", *args, stream=stream, sync=sync)
        return
    ptr, count, dtype, rows, cols, stride = _dense(x, "x", device, rows, cols, stride)
    packed = _checked_packed(codes, scales, rows, cols, device)
    _call("fe2o3_quantize_mxfp4", ptr, count, dtype, *packed, rows, cols, stride, stream=stream,
          sync=sync)


def dequantize_mxfp4(codes, scales, x, *, rows=None, cols=None, stride=None, stream=None,
                     sync=True) -> None:
    """The packed matrix's values into x, f32 or bf16 [rows, cols]
    (fe2o3_dequantize_mxfp4)."""
    device = _current_device()
    try:
        args = (_fast_packing(x, codes, scales, device)
                if rows is None and cols is None and stride is None else None)
    except _NOT_FAST:
        args = None
    if args is not None:
        _call("fe2o3_dequantize_mxfp4", *args[3:7], *args[:3], *args[7:], stream=stream, sync=sync)
        return
    ptr, count, dtype, rows, cols, stride = _dense(x, "x", device, rows, cols, stride)
    packed = _checked_packed(codes, scales, rows, cols, device)
    _call("fe2o3_dequantize_mxfp4", *packed, ptr, count, dtype, rows, cols, stride,
          stream=stream, sync=sync)


def _checked_packed(codes, scales, rows, cols, device):
    arrays, shapes = _packed(codes, scales, ("codes", "scales"), device)
    for name, found, want in zip(("codes", "scales"), shapes, mxfp4_shapes(rows, cols)):
        if found is not None and found != want:
            raise ValueError(f"{name} of {tuple(found)} for a matrix of {(rows, cols)}, not {want}")
    return arrays


def _fast_product(a, a_scales, b, b_scales, c, device):
    """The call's arguments, of tensors."""
    m, width = a.shape
    n, other = b.shape
    panels, a_rows, b_rows = width // 128, (m + 15) // 16 * 16, (n + 15) // 16 * 16
    a_at, b_at, c_at = _at(a, _is_bytes, device), _at(b, _is_bytes, device), _at(c, _is_bf16, device)
    as_at, bs_at = _at(a_scales, _is_bytes, device), _at(b_scales, _is_bytes, device)
    if (a_at is None or b_at is None or c_at is None or as_at is None or bs_at is None
            or width != other or width % 128 or a_scales.shape != (panels, a_rows, 8)
            or b_scales.shape != (panels, b_rows, 8) or c.shape != (m, n)):
        return None
    return (a_at, m * width, as_at, panels * a_rows * 8, b_at, n * width, bs_at,
            panels * b_rows * 8, c_at, m * n, m, n, panels * 256)


def gemm_mxfp4_nt(a, a_scales, b, b_scales, c, m=None, n=None, k=None, *, stream=None,
                  sync=True) -> None:
    """c (bf16 [m, n]) = A B^T of packed A [m, k] and B [n, k] (fe2o3_gemm_mxfp4_nt).  Sizes
    come from tensors (k in whole panels); DeviceBuffers take m, n, k."""
    device = _current_device()
    try:
        args = (_fast_product(a, a_scales, b, b_scales, c, device)
                if m is None and n is None and k is None else None)
    except _NOT_FAST:
        args = None
    if args is not None:
        _call("fe2o3_gemm_mxfp4_nt", *args, stream=stream, sync=sync)
        return
    left, (ca, sa) = _packed(a, a_scales, ("a", "a_scales"), device)
    right, (cb, sb) = _packed(b, b_scales, ("b", "b_scales"), device)
    shape = _dimensions(c, 2, "c")
    if ca is not None:
        found = (ca[0], cb[0] if cb is not None else n, 2 * ca[1])
        given = (m, n, k if k is None else -(-k // MXFP4_PANEL) * MXFP4_PANEL)
        if any(g is not None and g != f for g, f in zip(given, found)):
            raise ValueError(f"m, n, k of {(m, n, k)} for operands of {found}")
        m, n, k = found
    if m is None or n is None or k is None:
        raise ValueError("operands in DeviceBuffers need m, n and k")
    for name, found, want in (("a", ca, mxfp4_shapes(m, k)[0]), ("b", cb, mxfp4_shapes(n, k)[0]),
                              ("a_scales", sa, mxfp4_shapes(m, k)[1]),
                              ("b_scales", sb, mxfp4_shapes(n, k)[1]), ("c", shape, (m, n))):
        if found is not None and found != want:
            raise ValueError(f"{name} of {tuple(found)}, not {want}")
    _call("fe2o3_gemm_mxfp4_nt", *left, *right, *_operand(c, _BF16, "c", device), m, n, k,
          stream=stream, sync=sync)


def kernel_resources(entry: str) -> list[dict]:
    """Every kernel behind C-ABI entry point `entry` with its launch facts and
    the resources the runtime reports for the loaded code object
    (fe2o3_kernel_resources)."""
    L = _lib.lib()
    count = C.c_uint32(0)
    rc = L.fe2o3_kernel_resources(entry.encode(), 0xFFFFFFFF, None, C.byref(count))
    if rc not in (0, -2):
        check(rc, "fe2o3_kernel_resources")
    out = []
    for i in range(count.value):
        rec = _lib.Fe2o3KernelResources()
        check(L.fe2o3_kernel_resources(entry.encode(), i, C.byref(rec), C.byref(count)),
              "fe2o3_kernel_resources")
        out.append({name: (getattr(rec, name).decode() if name == "kernel" else getattr(rec, name))
                    for name, _ in rec._fields_})
    return out


def fill_normal_bf16(buf: DeviceBuffer, seed: int, domain: int, scale: float, first: int = 0,
                     stream=None, sync=True) -> None:
    _call("fe2o3_fill_normal_bf16", buf.ptr, buf.count, seed, domain, scale, first,
          stream=stream, sync=sync)


def fill_normal_f32(buf: DeviceBuffer, seed: int, domain: int, scale: float, first: int = 0,
                    stream=None, sync=True) -> None:
    _call("fe2o3_fill_normal_f32", buf.ptr, buf.count, seed, domain, scale, first,
          stream=stream, sync=sync)


def fill_uniform_f32(buf: DeviceBuffer, seed: int, domain: int, first: int = 0, stream=None,
                     sync=True) -> None:
    _call("fe2o3_fill_uniform_f32", buf.ptr, buf.count, seed, domain, first, stream=stream,
          sync=sync)
