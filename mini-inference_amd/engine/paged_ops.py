"""Tensor-level entry points of the paged KV-cache kernels.

Each function validates shapes on the host, then passes raw device pointers, element
strides and the current HIP stream through the C ABI (``include/mipaged.h``). Nothing
here computes on the CPU: tensors that are not on a ROCm device raise.
"""

from __future__ import annotations

import ctypes
import math
from functools import lru_cache
from itertools import chain

import numpy as np
import torch

from . import _native

MAX_TREE_NODES = _native.MIP_TREE_MAX_NODES

_DTYPE_CODES = {torch.float32: _native.MIP_F32, torch.float16: _native.MIP_F16, torch.bfloat16: _native.MIP_BF16}


def dtype_code(dtype: torch.dtype) -> int:
    try:
        return _DTYPE_CODES[dtype]
    except KeyError:
        raise TypeError(f"unsupported KV dtype {dtype}; expected float32, float16 or bfloat16") from None


def _require_device(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if not t.is_cuda:
            raise RuntimeError(
                "the paged KV-cache kernels run only on a ROCm GPU device (got a tensor on "
                f"{t.device}); there is no CPU path"
            )


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_ptr(device: torch.device) -> int:
    """Handle of the current stream on ``device`` (``torch.cuda.current_stream(device).cuda_stream``)."""
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


class PreparedCall:
    """One validated C-ABI call with its argument tuple fixed (pointers, strides, stream).

    Calling it re-launches the kernel on the same buffers with no Python-side checks, for
    loops over static buffers (timing, serving loops). The stream is the one current when
    the call was prepared: a call meant for a graph must be prepared inside the capture.
    The tensors passed to the ``prepare_*`` function must stay alive and in place while it
    is used.
    """

    __slots__ = ("_fn", "_args", "_what", "keep")

    def __init__(self, fn, args: tuple, what: str, keep: tuple = ()) -> None:
        self._fn, self._args, self._what, self.keep = fn, args, what, keep

    def __call__(self) -> None:
        st = self._fn(*self._args)
        if st:
            _native.check(st, self._what)


def _noop() -> None:
    return None


def prepare_kv_append(k_cache: torch.Tensor, v_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      slot_mapping: torch.Tensor):
    """Validate a :func:`kv_append` call once; returns a :class:`PreparedCall` (or a no-op for N = 0)."""
    _require_device(k_cache, v_cache, k, v, slot_mapping)
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache/v_cache must be contiguous [num_blocks, Hkv, block_size, D] tensors of one shape")
    nb, hkv, bs, d = k_cache.shape
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (hkv, d):
        raise ValueError(f"k/v must be [N, {hkv}, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != k_cache.dtype or v.dtype != k_cache.dtype or v_cache.dtype != k_cache.dtype:
        raise TypeError("k, v and the cache must share one dtype")
    if k.stride(2) != 1 or v.stride(2) != 1:
        raise ValueError("the last (head_dim) dimension of k/v must be contiguous")
    if slot_mapping.dtype != torch.int64 or slot_mapping.dim() != 1 or slot_mapping.shape[0] != k.shape[0]:
        raise ValueError("slot_mapping must be int64 [N]")
    if not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous")
    n = k.shape[0]
    if n == 0:
        return _noop
    lib = _native.load()
    args = (k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1),
            k_cache.data_ptr(), v_cache.data_ptr(), nb, slot_mapping.data_ptr(), n, hkv, d, bs,
            dtype_code(k_cache.dtype), _stream_ptr(k_cache.device))
    return PreparedCall(lib.mip_kv_append, args, "mip_kv_append", (k_cache, v_cache, k, v, slot_mapping))


def kv_append(k_cache: torch.Tensor, v_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              slot_mapping: torch.Tensor) -> None:
    """Write token i's K/V rows (``k[i, h, :]``) to pool slot ``slot_mapping[i]``.

    ``k_cache``/``v_cache``: one layer of the pool, ``[num_blocks + 1, Hkv, block_size, D]``
    contiguous. ``k``/``v``: ``[N, Hkv, D]`` with any token/head strides and a contiguous
    last dimension. ``slot_mapping``: int64 ``[N]``, ``block * block_size + offset``.
    Follows engine/kv_cache.py:613-614 and :286-289 (bit-exact data movement).
    """
    prepare_kv_append(k_cache, v_cache, k, v, slot_mapping)()


def prepare_rope_kv_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                           sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           slot_mapping: torch.Tensor):
    """Validate a :func:`rope_kv_append` call once; returns a :class:`PreparedCall` (or a no-op for N = 0)."""
    _require_device(k, v, cos, sin, k_cache, v_cache, slot_mapping)
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache/v_cache must be contiguous [num_blocks, Hkv, block_size, D] tensors of one shape")
    nb, hkv, bs, d = k_cache.shape
    if d % 2:
        raise ValueError(f"rotary embedding needs an even head_dim, got {d}")
    if k.dim() != 3 or k.shape != v.shape or k.shape[1:] != (hkv, d):
        raise ValueError(f"k/v must be [N, {hkv}, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    n = k.shape[0]
    if q is not None:
        _require_device(q)
        if q.dim() != 3 or q.shape[0] != n or q.shape[2] != d or q.stride(2) != 1:
            raise ValueError(f"q must be [{n}, Hq, {d}] with a contiguous last dimension, got {tuple(q.shape)}")
    if cos.shape != (n, d) or sin.shape != (n, d) or cos.stride() != sin.stride() or cos.stride(1) != 1:
        raise ValueError(f"cos/sin must be [{n}, {d}] with one stride and a contiguous last dimension")
    dt = k_cache.dtype
    if any(t.dtype != dt for t in (k, v, cos, sin, v_cache) + ((q,) if q is not None else ())):
        raise TypeError("q, k, v, cos, sin and the cache must share one dtype")
    if k.stride(2) != 1 or v.stride(2) != 1:
        raise ValueError("the last (head_dim) dimension of k/v must be contiguous")
    if slot_mapping.dtype != torch.int64 or slot_mapping.dim() != 1 or slot_mapping.shape[0] != n:
        raise ValueError("slot_mapping must be int64 [N]")
    if not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous")
    if n == 0:
        return _noop
    lib = _native.load()
    hq = 0 if q is None else q.shape[1]
    qp, qs0, qs1 = (None, 0, 0) if q is None else (q.data_ptr(), q.stride(0), q.stride(1))
    args = (qp, qs0, qs1, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
            cos.data_ptr(), sin.data_ptr(), cos.stride(0), k_cache.data_ptr(), v_cache.data_ptr(), nb,
            slot_mapping.data_ptr(), n, hq, hkv, d, bs, dtype_code(dt), _stream_ptr(k_cache.device))
    return PreparedCall(lib.mip_rope_kv_append, args, "mip_rope_kv_append",
                        (q, k, v, cos, sin, k_cache, v_cache, slot_mapping))


def rope_kv_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                   k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Rotate q and k in place (rotary embedding) and append the rotated k and v to the pool.

    ``q``: ``[N, Hq, D]`` (or None), ``k``/``v``: ``[N, Hkv, D]``, any token/head strides and a
    contiguous last dimension; ``cos``/``sin``: ``[N, D]`` rows per token. The values equal
    engine/model.py:216-224 (``x * cos + rotate_half(x) * sin`` evaluated op by op in the
    dtype) bit for bit, and the pool rows equal :func:`kv_append` of the rotated k and v.
    """
    prepare_rope_kv_append(q, k, v, cos, sin, k_cache, v_cache, slot_mapping)()


class _Workspace:
    """One scratch buffer per device, grown on demand (no initialisation needed).

    Calls that use it must be ordered (one stream, or graph replays on that stream): two
    decode calls running concurrently on different streams of one device would race on
    it; pass ``workspace=`` to each instead. A buffer that has been handed out is never
    freed: a captured graph may hold its address, so growing the workspace keeps the old
    buffer alive (``retired``) for the life of the process.
    """

    def __init__(self) -> None:
        self._bufs: dict[int, torch.Tensor] = {}
        self.retired: list[torch.Tensor] = []

    def get(self, device: torch.device, nbytes: int) -> torch.Tensor | None:
        if nbytes == 0:
            return None
        key = device.index if device.index is not None else torch.cuda.current_device()
        buf = self._bufs.get(key)
        if buf is None or buf.numel() < nbytes:
            if buf is not None:
                self.retired.append(buf)
            size = max(nbytes, 2 * buf.numel() if buf is not None else 0)
            buf = torch.empty(size, dtype=torch.uint8, device=device)
            self._bufs[key] = buf
        return buf


_workspace = _Workspace()


def decode_workspace_bytes(batch: int, num_heads: int, num_kv_heads: int, head_dim: int, block_size: int,
                           max_blocks: int, dtype: torch.dtype) -> int:
    """Bytes of scratch a decode call of this shape needs (``mip_paged_decode_workspace``)."""
    return int(_native.load().mip_paged_decode_workspace(batch, num_heads, num_kv_heads, head_dim, block_size,
                                                         max_blocks, dtype_code(dtype)))


def _plan_key(batch: int, num_heads: int, num_kv_heads: int, head_dim: int, block_size: int, max_blocks: int,
              dtype: torch.dtype) -> tuple:
    """The shape a work plan is laid out for (its tensor carries it as ``_mip_plan_key``)."""
    return (batch, num_heads, num_kv_heads, head_dim, block_size, max_blocks, dtype)


def prepare_paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                         context_lens: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None,
                         max_blocks: int | None = None, workspace: torch.Tensor | None = None,
                         append: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
                         plan: torch.Tensor | None = None):
    """Validate a :func:`paged_decode` call once; returns ``(PreparedCall, out)``.

    ``append = (k, v, slot_mapping)`` prepares the fused append + decode call
    (:func:`paged_decode_append`) instead. ``plan`` is a work plan from :func:`decode_plan`
    for the same context lengths and block tables (or None).
    """
    _require_device(q, k_cache, v_cache, block_tables, context_lens)
    if q.dim() != 3 or q.stride(2) != 1:
        raise ValueError("q must be [B, Hq, D] with a contiguous last dimension")
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache/v_cache must be contiguous [num_blocks, Hkv, block_size, D] tensors of one shape")
    nb, hkv, bs, d = k_cache.shape
    b, hq, dq = q.shape
    if dq != d or hq % hkv != 0:
        raise ValueError(f"q {tuple(q.shape)} does not match the cache (Hkv={hkv}, D={d})")
    if q.dtype != k_cache.dtype or v_cache.dtype != k_cache.dtype:
        raise TypeError("q and the cache must share one dtype")
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.shape[0] != b:
        raise ValueError("block_tables must be int32 [B, max_blocks]")
    if block_tables.stride(1) != 1:
        raise ValueError("block_tables rows must be contiguous")
    if context_lens.dtype != torch.int32 or context_lens.shape != (b,) or not context_lens.is_contiguous():
        raise ValueError("context_lens must be contiguous int32 [B]")
    mb = block_tables.shape[1] if max_blocks is None else int(max_blocks)
    if mb < 1 or mb > block_tables.shape[1]:
        raise ValueError(f"max_blocks={mb} is outside [1, {block_tables.shape[1]}]")
    if out is None:
        out = torch.empty((b, hq, d), dtype=q.dtype, device=q.device)
    elif out.shape != (b, hq, d) or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError("out must be [B, Hq, D] in q's dtype with a contiguous last dimension")
    if b == 0:
        return _noop, out
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    code = dtype_code(q.dtype)
    lib = _native.load()
    need = int(lib.mip_paged_decode_workspace(b, hq, hkv, d, bs, mb, code))
    if workspace is None:
        workspace = _workspace.get(q.device, need)
    elif need and workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace holds {workspace.numel() * workspace.element_size()} bytes, needs {need}")
    ws_ptr = workspace.data_ptr() if workspace is not None else None
    ws_bytes = workspace.numel() * workspace.element_size() if workspace is not None else 0
    if plan is not None:
        _require_device(plan)
        if plan.dtype != torch.int32 or not plan.is_contiguous():
            raise ValueError("plan must be a contiguous int32 tensor from decode_plan")
        made_for = getattr(plan, "_mip_plan_key", None)
        want = _plan_key(b, hq, hkv, d, bs, mb, q.dtype)
        if made_for is not None and made_for != want:
            raise ValueError(f"the plan was made for shape {made_for}, not this call's {want}")
    plan_ptr = plan.data_ptr() if plan is not None else None
    plan_bytes = plan.numel() * 4 if plan is not None else 0
    args = (out.data_ptr(), out.stride(0), out.stride(1), q.data_ptr(), q.stride(0), q.stride(1),
            k_cache.data_ptr(), v_cache.data_ptr(), nb, block_tables.data_ptr(), block_tables.stride(0),
            context_lens.data_ptr(), b, hq, hkv, d, bs, mb, scale, ws_ptr, ws_bytes, plan_ptr, plan_bytes, code,
            _stream_ptr(q.device))
    keep = (out, q, k_cache, v_cache, block_tables, context_lens, workspace, plan)  # [4:8]: the step's
    if append is None:
        return PreparedCall(lib.mip_paged_decode, args, "mip_paged_decode", keep), out
    k, v, slot_mapping = append
    _require_device(k, v, slot_mapping)
    if k.shape != (b, hkv, d) or v.shape != (b, hkv, d):
        raise ValueError(f"k/v must be [{b}, {hkv}, {d}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dtype != k_cache.dtype or v.dtype != k_cache.dtype:
        raise TypeError("k, v and the cache must share one dtype")
    if k.stride(2) != 1 or v.stride(2) != 1:
        raise ValueError("the last (head_dim) dimension of k/v must be contiguous")
    if slot_mapping.dtype != torch.int64 or slot_mapping.shape != (b,) or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous int64 [B]")
    fused = (k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0), v.stride(1), slot_mapping.data_ptr(),
             *args)
    return PreparedCall(lib.mip_paged_decode_append, fused, "mip_paged_decode_append", keep + (k, v, slot_mapping)), out


def _layout(t: torch.Tensor) -> tuple:
    return (t.shape, t.stride(), t.dtype, t.device)


class _LayerCalls:
    """The per-layer calls of one step, with what the layers share checked and laid out once.

    Within a step every layer's call takes the same tables, lengths, slots and sizes; only the
    layer's tensors change, and they keep one layout. The first call of a kind runs the full checks
    (the ``prepare_*`` functions) and keeps their arguments as a struct of the C ABI; a later call
    whose tensors have the same layout (shapes, strides, dtypes, devices) passes that struct, the
    new addresses and the current stream. Any other call is checked in full again.

    Tensors come as an attention layer has them, ``[B, H, T, D]``, and pools whole,
    ``[L, num_blocks + 1, Hkv, block_size, D]``.
    """

    def __init__(self) -> None:
        # kind -> (layout key, address of the struct, layers, K and V layer bytes, the struct, kept tensors)
        self._cached: dict[str, tuple] = {}

    def _hit(self, kind: str, key: tuple, layer) -> tuple | None:
        hit = self._cached.get(kind)
        if hit is None or hit[0] != key or type(layer) is not int or not 0 <= layer < hit[2]:
            return None
        return hit

    def _keep(self, kind: str, key: tuple, step, k_pool: torch.Tensor, v_pool: torch.Tensor, keep: tuple) -> None:
        # keep: the tensors that the struct points to, and none of a layer's own.
        self._cached[kind] = (key, ctypes.addressof(step), min(k_pool.shape[0], v_pool.shape[0]),
                              k_pool.stride(0) * k_pool.element_size(), v_pool.stride(0) * v_pool.element_size(), step,
                              keep)


class DecodeStepCalls(_LayerCalls):
    """The layer calls of one decode step (one token per sequence). ``plan`` maps (num_heads, dtype) to the
    step's work plan (or None)."""

    def __init__(self, block_tables: torch.Tensor, context_lens: torch.Tensor, slot_mapping: torch.Tensor,
                 scale: float, max_blocks: int, plan) -> None:
        super().__init__()
        self.block_tables, self.context_lens, self.slot_mapping = block_tables, context_lens, slot_mapping
        self.scale, self.max_blocks, self._plan = scale, max_blocks, plan

    def append_attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor,
                      v_pool: torch.Tensor) -> torch.Tensor:
        """:func:`paged_decode_append` of one layer; returns ``[B, Hq, 1, D]``."""
        key = (_layout(q), _layout(k), _layout(v), _layout(k_pool), _layout(v_pool))
        hit = self._hit("append", key, layer)
        if hit is not None:
            _, step, _, kb, vb, _, _ = hit
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            st = _native.load().mip_decode_step_append(step, k.data_ptr(), v.data_ptr(), out.data_ptr(), q.data_ptr(),
                                                       k_pool.data_ptr() + layer * kb, v_pool.data_ptr() + layer * vb,
                                                       _stream_ptr(q.device))
            if st:
                _native.check(st, "mip_decode_step_append")
            return out
        q1 = q[:, :, 0]
        call, out = prepare_paged_decode(q1, k_pool[layer], v_pool[layer], self.block_tables, self.context_lens,
                                         self.scale, None, self.max_blocks, append=(k[:, :, 0], v[:, :, 0],
                                                                                    self.slot_mapping),
                                         plan=self._plan(q1.shape[1], q1.dtype))
        call()
        if call is not _noop and q.shape[2] == k.shape[2] == v.shape[2] == 1:
            a = call._args
            self._keep("append", key, self._struct(a[7:], a[2:6], a[6]), k_pool, v_pool,
                       (self.slot_mapping, *call.keep[4:8]))
        return out.unsqueeze(2)

    def attend(self, layer: int, q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor) -> torch.Tensor:
        """:func:`paged_decode` of one layer; returns ``[B, Hq, 1, D]``."""
        key = (_layout(q), _layout(k_pool), _layout(v_pool))
        hit = self._hit("decode", key, layer)
        if hit is not None:
            _, step, _, kb, vb, _, _ = hit
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            st = _native.load().mip_decode_step_attend(step, out.data_ptr(), q.data_ptr(),
                                                       k_pool.data_ptr() + layer * kb, v_pool.data_ptr() + layer * vb,
                                                       _stream_ptr(q.device))
            if st:
                _native.check(st, "mip_decode_step_attend")
            return out
        q1 = q[:, :, 0]
        call, out = prepare_paged_decode(q1, k_pool[layer], v_pool[layer], self.block_tables, self.context_lens,
                                         self.scale, None, self.max_blocks, plan=self._plan(q1.shape[1], q1.dtype))
        call()
        if call is not _noop and q.shape[2] == 1:
            self._keep("decode", key, self._struct(call._args, (0, 0, 0, 0), None), k_pool, v_pool, call.keep[4:8])
        return out.unsqueeze(2)

    @staticmethod
    def _struct(a: tuple, kv_strides: tuple, slots) -> _native.DecodeStep:
        # a: the arguments of mip_paged_decode
        return _native.DecodeStep(*kv_strides, slots, a[1], a[2], a[4], a[5], a[8], a[9], a[10], a[11], a[19], a[20],
                                  a[21], a[22], *a[12:18], a[23], a[18])

    def rope_append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                    sin: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor) -> None:
        """:func:`rope_kv_append` of one layer (q and k rotated in place); cos, sin ``[B, 1, 1, D]``."""
        key = (_layout(q), _layout(k), _layout(v), _layout(cos), _layout(sin), _layout(k_pool), _layout(v_pool))
        if _rope_hit(self, layer, key, q, k, v, cos, sin, k_pool, v_pool):
            return
        call = prepare_rope_kv_append(q[:, :, 0], k[:, :, 0], v[:, :, 0], cos[:, 0, 0], sin[:, 0, 0], k_pool[layer],
                                      v_pool[layer], self.slot_mapping)
        call()
        if call is not _noop and all(t.shape[2] == 1 for t in (q, k, v)):
            self._keep("rope", key, _rope_struct(call._args), k_pool, v_pool, (self.slot_mapping,))


def _rope_hit(calls: _LayerCalls, layer, key, q, k, v, cos, sin, k_pool, v_pool) -> bool:
    hit = calls._hit("rope", key, layer)
    if hit is None:
        return False
    _, step, _, kb, vb, _, _ = hit
    st = _native.load().mip_rope_step_append(step, q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(),
                                             sin.data_ptr(), k_pool.data_ptr() + layer * kb,
                                             v_pool.data_ptr() + layer * vb, _stream_ptr(k.device))
    if st:
        _native.check(st, "mip_rope_step_append")
    return True


def _rope_struct(a: tuple) -> _native.RopeStep:
    # a: the arguments of mip_rope_kv_append
    return _native.RopeStep(a[1], a[2], a[4], a[5], a[7], a[8], a[11], a[14], a[15], *a[16:22])


class PrefillStepCalls(_LayerCalls):
    """The layer calls of one packed prefill step; q, k, v ``[1, H, N, D]``, cos and sin ``[1, 1, N, D]``."""

    def __init__(self, block_tables: torch.Tensor, cu_q: torch.Tensor, ctx_start: torch.Tensor,
                 slot_mapping: torch.Tensor, max_q_len: int, scale: float) -> None:
        super().__init__()
        self.block_tables, self.cu_q, self.ctx_start, self.slot_mapping = block_tables, cu_q, ctx_start, slot_mapping
        self.max_q_len, self.scale = max_q_len, scale

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor) -> None:
        """:func:`kv_append` of one layer's new tokens."""
        key = (_layout(k), _layout(v), _layout(k_pool), _layout(v_pool))
        hit = self._hit("append", key, layer)
        if hit is not None:
            _, step, _, kb, vb, _, _ = hit
            st = _native.load().mip_prefill_step_append(step, k.data_ptr(), v.data_ptr(), k_pool.data_ptr() + layer * kb,
                                                        v_pool.data_ptr() + layer * vb, _stream_ptr(k_pool.device))
            if st:
                _native.check(st, "mip_prefill_step_append")
            return
        # k[0] is [Hkv, N, D]; the append kernel takes [N, Hkv, D] views with any strides.
        call = prepare_kv_append(k_pool[layer], v_pool[layer], k[0].transpose(0, 1), v[0].transpose(0, 1),
                                 self.slot_mapping)
        call()
        if call is not _noop and k.shape[0] == v.shape[0] == 1:
            a = call._args
            step = _native.PrefillStep(k_stride_tok=a[2], k_stride_head=a[3], v_stride_tok=a[4], v_stride_head=a[5],
                                       slot_mapping=a[9], num_cache_blocks=a[8], n_tokens=a[10], num_kv_heads=a[11],
                                       head_dim=a[12], block_size=a[13], dtype=a[14])
            self._keep("append", key, step, k_pool, v_pool, (self.slot_mapping,))

    def rope_append(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor,
                    sin: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor) -> None:
        """:func:`rope_kv_append` of one layer's new tokens (q and k rotated in place)."""
        key = (_layout(q), _layout(k), _layout(v), _layout(cos), _layout(sin), _layout(k_pool), _layout(v_pool))
        if _rope_hit(self, layer, key, q, k, v, cos, sin, k_pool, v_pool):
            return
        call = prepare_rope_kv_append(q[0].transpose(0, 1), k[0].transpose(0, 1), v[0].transpose(0, 1), cos[0, 0],
                                      sin[0, 0], k_pool[layer], v_pool[layer], self.slot_mapping)
        call()
        if call is not _noop and all(t.shape[0] == 1 for t in (q, k, v)):
            self._keep("rope", key, _rope_struct(call._args), k_pool, v_pool, (self.slot_mapping,))

    def attend(self, layer: int, q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor) -> torch.Tensor:
        """:func:`paged_prefill` of one layer; returns ``[1, Hq, N, D]``, a view of ``[N, Hq, D]``."""
        key = (_layout(q), _layout(k_pool), _layout(v_pool))
        hit = self._hit("attend", key, layer)
        if hit is not None:
            _, step, _, kb, vb, _, _ = hit
            _, hq, n, d = q.shape
            out = torch.empty_strided((1, hq, n, d), (hq * d, d, hq * d, 1), dtype=q.dtype, device=q.device)
            st = _native.load().mip_prefill_step_attend(step, out.data_ptr(), q.data_ptr(),
                                                        k_pool.data_ptr() + layer * kb, v_pool.data_ptr() + layer * vb,
                                                        _stream_ptr(q.device))
            if st:
                _native.check(st, "mip_prefill_step_attend")
            return out
        # q is [1, Hq, N, D]; the kernel takes the [N, Hq, D] view and returns [N, Hq, D].
        call, out = prepare_paged_prefill(q[0].transpose(0, 1), k_pool[layer], v_pool[layer], self.block_tables,
                                          self.cu_q, self.ctx_start, self.max_q_len, scale=self.scale)
        call()
        if q.shape[0] == 1 and q.shape[2] > 0:
            a = call._args
            step = _native.PrefillStep(out_stride_tok=a[1], out_stride_head=a[2], q_stride_tok=a[4], q_stride_head=a[5],
                                       num_cache_blocks=a[8], block_tables=a[9], bt_stride=a[10], cu_q=a[11],
                                       ctx_start=a[12], num_seqs=a[13], max_q_len=a[14], num_heads=a[15],
                                       num_kv_heads=a[16], head_dim=a[17], block_size=a[18], max_blocks_per_seq=a[19],
                                       scale=a[20], dtype=a[21])
            self._keep("attend", key, step, k_pool, v_pool, (self.block_tables, self.cu_q, self.ctx_start))
        return out.transpose(0, 1).unsqueeze(0)


def prepare_decode_plan(context_lens: torch.Tensor, block_tables: torch.Tensor, num_heads: int, num_kv_heads: int,
                        head_dim: int, block_size: int, dtype: torch.dtype, max_blocks: int | None = None,
                        plan: torch.Tensor | None = None):
    """A prepared :func:`decode_plan` launch and its plan tensor, or ``(None, None)`` where the
    stream kernel does not run (then decode calls take no plan)."""
    _require_device(context_lens, block_tables)
    if block_tables.dtype != torch.int32 or block_tables.dim() != 2 or block_tables.stride(1) != 1:
        raise ValueError("block_tables must be int32 [B, max_blocks] with contiguous rows")
    b = block_tables.shape[0]
    if context_lens.dtype != torch.int32 or context_lens.shape != (b,) or not context_lens.is_contiguous():
        raise ValueError("context_lens must be contiguous int32 [B]")
    mb = block_tables.shape[1] if max_blocks is None else int(max_blocks)
    code = dtype_code(dtype)
    lib = _native.load()
    need = int(lib.mip_paged_decode_plan_bytes(b, num_heads, num_kv_heads, head_dim, block_size, mb, code))
    if need == 0:
        return None, None
    if plan is None:
        plan = torch.empty(-(-need // 4), dtype=torch.int32, device=context_lens.device)
    elif plan.dtype != torch.int32 or not plan.is_contiguous() or plan.numel() * 4 < need:
        raise ValueError(f"plan must be a contiguous int32 tensor of at least {need} bytes")
    plan._mip_plan_key = _plan_key(b, num_heads, num_kv_heads, head_dim, block_size, mb, dtype)
    args = (context_lens.data_ptr(), block_tables.data_ptr(), block_tables.stride(0), b, num_heads, num_kv_heads,
            head_dim, block_size, mb, code, plan.data_ptr(), plan.numel() * 4, _stream_ptr(context_lens.device))
    keep = (context_lens, block_tables, plan)
    return PreparedCall(lib.mip_paged_decode_plan, args, "mip_paged_decode_plan", keep), plan


def decode_plan(context_lens: torch.Tensor, block_tables: torch.Tensor, num_heads: int, num_kv_heads: int,
                head_dim: int, block_size: int, dtype: torch.dtype, max_blocks: int | None = None,
                plan: torch.Tensor | None = None) -> torch.Tensor | None:
    """One decode step's work plan for the stream kernel (None where that kernel does not run).

    Every layer's :func:`paged_decode` / :func:`paged_decode_append` with these context
    lengths and tables can take it and skip deriving the work split.
    """
    call, plan = prepare_decode_plan(context_lens, block_tables, num_heads, num_kv_heads, head_dim, block_size,
                                     dtype, max_blocks, plan)
    if call is not None:
        call()
    return plan


def paged_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                 context_lens: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None,
                 max_blocks: int | None = None, workspace: torch.Tensor | None = None,
                 plan: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention over paged K/V for one query token per sequence.

    ``q``: ``[B, Hq, D]`` (last dim contiguous). ``k_cache``/``v_cache``: one layer,
    ``[num_blocks + 1, Hkv, block_size, D]``. ``block_tables``: int32 ``[B, >= max_blocks]``.
    ``context_lens``: int32 ``[B]`` (keys attended = positions + 1). Returns ``out``
    ``[B, Hq, D]`` in q's dtype. Follows engine/kv_cache.py:615-620 and
    engine/model.py:126-147 with ``scale = 1/sqrt(D)`` by default.
    """
    call, out = prepare_paged_decode(q, k_cache, v_cache, block_tables, context_lens, scale, out, max_blocks,
                                     workspace, plan=plan)
    call()
    return out


def decode_prepare(rows: torch.Tensor, journal_flat: torch.Tensor, journal_block: torch.Tensor, row_ids: torch.Tensor,
                   positions: torch.Tensor, tables: torch.Tensor, n_blocks: int, slot_mapping: torch.Tensor,
                   context_lens: torch.Tensor, block_size: int) -> None:
    """A decode step's inputs from the device mirror of the block tables (``mip_decode_prepare``): apply the journal
    to ``rows``, gather the batch's first ``n_blocks`` entries into ``tables``, and write each new token's slot and
    each sequence's length."""
    _require_device(rows, journal_flat, journal_block, row_ids, positions, tables, slot_mapping, context_lens)
    for t in (journal_flat, journal_block, row_ids, positions, slot_mapping):
        if t.dtype != torch.int64 or t.dim() != 1 or not t.is_contiguous():
            raise ValueError("journal, row ids, positions and slots must be contiguous int64 vectors")
    if rows.dtype != torch.int32 or not rows.is_contiguous() or tables.dtype != torch.int32 or tables.stride(1) != 1:
        raise ValueError("rows and tables must be int32 with contiguous rows")
    b = row_ids.shape[0]
    if (journal_flat.shape != journal_block.shape or positions.shape[0] != b or slot_mapping.shape[0] != b
            or context_lens.shape != (b,) or context_lens.dtype != torch.int32 or not context_lens.is_contiguous()
            or tables.shape[0] < b or min(tables.shape[1], rows.shape[1]) < n_blocks):
        raise ValueError("decode_prepare: the batch's tensors do not match")
    st = _native.load().mip_decode_prepare(rows.data_ptr(), rows.stride(0), journal_flat.data_ptr(),
                                           journal_block.data_ptr(), journal_flat.shape[0], row_ids.data_ptr(),
                                           positions.data_ptr(), tables.data_ptr(), tables.stride(0), n_blocks,
                                           slot_mapping.data_ptr(), context_lens.data_ptr(), b, block_size,
                                           _stream_ptr(rows.device))
    if st:
        _native.check(st, "mip_decode_prepare")


def prefill_index(cu_q: torch.Tensor, ctx_start: torch.Tensor, block_tables: torch.Tensor, n_tokens: int,
                  max_q_len: int, block_size: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``positions`` and ``slot_mapping`` (int64 ``[n_tokens]``) of a packed prefill step's new tokens, and
    ``last_index`` (int64 ``[S]``), from the tensors :func:`paged_prefill` takes. Follows
    engine/kv_cache.py:230-250, 562-573.
    """
    if not cu_q.dtype == ctx_start.dtype == block_tables.dtype == torch.int32:
        raise ValueError("cu_q, ctx_start and block_tables must be int32")
    s = ctx_start.numel()
    if (ctx_start.dim() != 1 or cu_q.dim() != 1 or cu_q.numel() != s + 1 or block_tables.dim() != 2
            or block_tables.size(0) < s or n_tokens < 0 or max_q_len < 0):
        raise ValueError("prefill_index: the step's tensors do not match")
    if not (cu_q.is_contiguous() and ctx_start.is_contiguous()) or block_tables.stride(1) != 1:
        raise ValueError("cu_q, ctx_start and the block_tables rows must be contiguous")
    _require_device(cu_q, ctx_start, block_tables)
    out = torch.empty(2 * n_tokens + s, dtype=torch.int64, device=cu_q.device)
    positions, slots, last = out[:n_tokens], out[n_tokens:2 * n_tokens], out[2 * n_tokens:]
    if s:
        st = _native.load().mip_prefill_index(positions.data_ptr(), slots.data_ptr(), last.data_ptr(), cu_q.data_ptr(),
                                              ctx_start.data_ptr(), block_tables.data_ptr(), block_tables.stride(0), s,
                                              max_q_len, block_size, _stream_ptr(cu_q.device))
        if st:
            _native.check(st, "mip_prefill_index")
    return positions, slots, last


def prepare_paged_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                          cu_q: torch.Tensor, ctx_start: torch.Tensor, max_q_len: int, scale: float | None = None,
                          out: torch.Tensor | None = None, max_blocks: int | None = None):
    """Validate a :func:`paged_prefill` call once; returns ``(PreparedCall, out)``."""
    _require_device(q, k_cache, v_cache, block_tables, cu_q, ctx_start)
    if q.dim() != 3 or q.stride(2) != 1:
        raise ValueError("q must be [N, Hq, D] with a contiguous last dimension")
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache/v_cache must be contiguous [num_blocks, Hkv, block_size, D] tensors of one shape")
    nb1, hkv, bs, d = k_cache.shape
    n, hq, dq = q.shape
    if dq != d or hq % hkv:
        raise ValueError(f"q {tuple(q.shape)} does not match the pool (Hkv={hkv}, D={d})")
    if q.dtype != k_cache.dtype or v_cache.dtype != k_cache.dtype:
        raise TypeError("q and the cache must share one dtype")
    if block_tables.dtype != torch.int32 or cu_q.dtype != torch.int32 or ctx_start.dtype != torch.int32:
        raise TypeError("block_tables, cu_q and ctx_start must be int32")
    num_seqs = ctx_start.shape[0]
    if block_tables.dim() != 2 or block_tables.shape[0] < num_seqs or block_tables.stride(1) != 1:
        raise ValueError("block_tables must be [S, nb] with contiguous rows")
    if cu_q.shape != (num_seqs + 1,) or not (cu_q.is_contiguous() and ctx_start.is_contiguous()):
        raise ValueError("cu_q must be int32 [S + 1] and ctx_start int32 [S], contiguous")
    nbm = block_tables.shape[1] if max_blocks is None else max_blocks
    if out is None:
        out = torch.empty(n, hq, d, dtype=q.dtype, device=q.device)
    elif out.shape != (n, hq, d) or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError("out must be [N, Hq, D] in q's dtype with a contiguous last dimension")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    lib = _native.load()
    args = (out.data_ptr(), out.stride(0), out.stride(1), q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(),
            v_cache.data_ptr(), nb1, block_tables.data_ptr(), block_tables.stride(0), cu_q.data_ptr(),
            ctx_start.data_ptr(), num_seqs, max_q_len, hq, hkv, d, bs, nbm, scale, dtype_code(q.dtype),
            _stream_ptr(q.device))
    keep = (out, q, k_cache, v_cache, block_tables, cu_q, ctx_start)
    return PreparedCall(lib.mip_paged_prefill, args, "mip_paged_prefill", keep), out


def paged_prefill(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                  cu_q: torch.Tensor, ctx_start: torch.Tensor, max_q_len: int, scale: float | None = None,
                  out: torch.Tensor | None = None, max_blocks: int | None = None) -> torch.Tensor:
    """Varlen causal attention of packed new tokens over their sequences' paged keys.

    ``q``: ``[N, Hq, D]`` packed rows (last dim contiguous); sequence ``s`` owns rows
    ``cu_q[s] .. cu_q[s+1]-1`` (int32 ``[S+1]``), at positions ``ctx_start[s] + i``
    (int32 ``[S]``), and each row attends its sequence's keys ``0 .. position`` read from the
    pool through ``block_tables`` (int32 ``[S, >= max_blocks]``). Returns ``out [N, Hq, D]``.
    Follows engine/kv_cache.py:268-294 (prefix read-back + mask) and :290-294 (packed causal).
    16-bit data at head_dim 64/128 runs the MFMA prefill kernel, fp32 at those sizes the fp32 MFMA
    kernel where it pays (up to 16 query heads per kv head each), other shapes (power-of-two head sizes 8 to
    256) the VALU kernel; anything else raises.
    """
    call, out = prepare_paged_prefill(q, k_cache, v_cache, block_tables, cu_q, ctx_start, max_q_len, scale, out,
                                      max_blocks)
    call()
    return out


def paged_decode_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                        v_cache: torch.Tensor, slot_mapping: torch.Tensor, block_tables: torch.Tensor,
                        context_lens: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None,
                        max_blocks: int | None = None, workspace: torch.Tensor | None = None,
                        plan: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`kv_append` of the step's ``k``/``v`` ``[B, Hkv, D]`` at ``slot_mapping``, then
    :func:`paged_decode`, as one call (engine/kv_cache.py:611-620). One kernel launch on the
    stream-kernel path; ``slot_mapping[b]`` must be the slot of key ``context_lens[b] - 1``
    (or outside the pool).
    """
    call, out = prepare_paged_decode(q, k_cache, v_cache, block_tables, context_lens, scale, out, max_blocks,
                                     workspace, append=(k, v, slot_mapping), plan=plan)
    call()
    return out


def _copy_shape(k_pool: torch.Tensor, v_pool: torch.Tensor) -> tuple[int, int, int]:
    if k_pool.shape != v_pool.shape or k_pool.dim() != 5 or not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError("k_pool/v_pool must be contiguous [L, num_blocks, Hkv, block_size, D] tensors of one shape")
    layers, blocks, heads, block_size, dim = k_pool.shape
    if layers == 0 or blocks == 0:
        raise IndexError("the pool holds no blocks")
    return layers, blocks, heads * block_size * dim * k_pool.element_size()


def _host_pairs(pairs) -> np.ndarray:
    """A private contiguous int64 [n, 2] copy of ``pairs`` (a CPU tensor, an array or a
    sequence of (src, dst)), so a prepared call keeps the pairs it was prepared with."""
    if isinstance(pairs, torch.Tensor):
        pairs = pairs.numpy()
    elif type(pairs) is list and set(map(type, pairs)) == {tuple} and set(map(len, pairs)) == {2}:
        # What prepare_writes builds: read flat, a third of the time of the nested conversion.
        return np.fromiter(chain.from_iterable(pairs), np.int64, 2 * len(pairs)).reshape(-1, 2)
    return np.array(pairs, dtype=np.int64, copy=True, order="C").reshape(-1, 2)


def prepare_copy_blocks(k_pool: torch.Tensor, v_pool: torch.Tensor, pairs):
    """Validate a :func:`copy_blocks` call once; returns a :class:`PreparedCall` (or a no-op for no pairs).

    ``pairs`` on the pool's device: ``mip_copy_blocks`` reads them from device memory (a
    graph replay sees later writes to that tensor). Anything else (a CPU tensor, an array, a
    sequence of (src, dst)): ``mip_copy_blocks_host`` passes them in the kernel arguments, as
    they are when the call is prepared.
    """
    _require_device(k_pool, v_pool)
    num_layers, nb, block_bytes = _copy_shape(k_pool, v_pool)
    stream = _stream_ptr(k_pool.device)
    if isinstance(pairs, torch.Tensor) and pairs.is_cuda:
        _require_device(pairs)
        if pairs.dtype != torch.int64 or pairs.dim() != 2 or pairs.shape[1] != 2 or not pairs.is_contiguous():
            raise ValueError("pairs must be contiguous int64 [n, 2]")
        if pairs.device != k_pool.device:
            raise ValueError("pairs on a device must be on the pool's device")
        n = pairs.shape[0]
        if n == 0:
            return _noop
        args = (k_pool.data_ptr(), v_pool.data_ptr(), pairs.data_ptr(), n, num_layers, nb, block_bytes, stream)
        return PreparedCall(_native.load().mip_copy_blocks, args, "mip_copy_blocks", (k_pool, v_pool, pairs))
    arr = _host_pairs(pairs)
    n = arr.shape[0]
    if n == 0:
        return _noop
    args = (k_pool.data_ptr(), v_pool.data_ptr(), arr.ctypes.data, n, num_layers, nb, block_bytes, stream)
    return PreparedCall(_native.load().mip_copy_blocks_host, args, "mip_copy_blocks_host", (k_pool, v_pool, arr))


def copy_blocks(k_pool: torch.Tensor, v_pool: torch.Tensor, pairs) -> None:
    """Copy whole blocks, every layer, K and V: ``pool[:, dst] = pool[:, src]`` per (src, dst) row.

    ``k_pool``/``v_pool``: ``[num_layers, num_blocks + 1, Hkv, block_size, D]`` contiguous.
    ``pairs``: int64 ``[n, 2]`` on the pool's device, or (src, dst) pairs on the host (a CPU
    tensor, an array or a sequence), which travel in the kernel arguments with no upload.
    Bitwise copy (no reference counterpart; used for copy-on-write of shared prefix blocks).
    """
    prepare_copy_blocks(k_pool, v_pool, pairs)()


def _one_device(*tensors: torch.Tensor) -> torch.device:
    """The device that all of these are on; a call whose pointers belong to several is refused."""
    device, index = tensors[0].device, tensors[0].get_device()
    for t in tensors:
        if t.get_device() != index or (index < 0 and t.device != device):
            raise ValueError(f"tensors on different devices: {device} and {t.device}")
    if not tensors[0].is_cuda:
        _require_device(tensors[0])
    return device


def _call_on(device: torch.device, fn, args: tuple, what: str) -> None:
    """Launch on the current stream of ``device``, whichever device is current."""
    if device.index == torch.cuda.current_device():
        st = fn(*args, _stream_ptr(device))
    else:
        with torch.cuda.device(device):
            st = fn(*args, _stream_ptr(device))
    if st:
        _native.check(st, what)


_I32 = torch.int32


def _tree_rows(cu_q: torch.Tensor, block_tables: torch.Tensor, ctx_start: torch.Tensor, max_q_len: int,
               max_blocks: int | None) -> tuple[int, int]:
    """Check the tensors that describe a step of trees; returns (sequences, blocks of a table)."""
    if not cu_q.dtype == ctx_start.dtype == block_tables.dtype == _I32:
        raise TypeError("cu_q, ctx_start and block_tables must be int32")
    seqs, tab = ctx_start.shape, block_tables.shape
    if len(seqs) != 1 or cu_q.shape != (seqs[0] + 1,):
        raise ValueError("cu_q must be int32 [S + 1] and ctx_start int32 [S]")
    s = seqs[0]
    if len(tab) != 2 or tab[0] < s or tab[1] < 1:
        raise ValueError("block_tables must be int32 [S, max_blocks]")
    if not (cu_q.is_contiguous() and ctx_start.is_contiguous()) or block_tables.stride(1) != 1:
        raise ValueError("cu_q, ctx_start and the block_tables rows must be contiguous")
    if max_q_len < 0:
        raise ValueError(f"max_q_len={max_q_len} is negative")
    mb = tab[1] if max_blocks is None else int(max_blocks)
    if mb < 1 or mb > tab[1]:
        raise ValueError(f"max_blocks={mb} is outside [1, {tab[1]}]")
    return s, mb


def _scratch(workspace: torch.Tensor | None, device: torch.device, need: int) -> torch.Tensor | None:
    """A call's scratch memory: the caller's, or new memory from the current stream's allocator.

    The latter is the call's own: calls on several streams and captured graphs (whose private pool it comes from) do
    not meet in it, and the allocator hands it on only behind the call's kernels on its stream."""
    if workspace is None:
        return torch.empty(need, dtype=torch.uint8, device=device) if need else None
    if need and workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace holds {workspace.numel() * workspace.element_size()} bytes, needs {need}")
    if workspace.device != device or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous tensor on the call's device")
    return workspace


def _extent(workspace: torch.Tensor | None) -> tuple[int | None, int]:
    """Address and size of scratch memory."""
    return (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel() * workspace.element_size())


@lru_cache(4096)
def _tree_bytes(device: torch.device, *shape) -> int:
    with torch.cuda.device(device):  # the size follows the current device
        return int(_native.load().mip_paged_tree_workspace(*shape))


@lru_cache(4096)
def _verify_bytes(*shape) -> int:
    return int(_native.load().mip_tree_verify_workspace(*shape))


def tree_index(parents: torch.Tensor, cu_q: torch.Tensor, ctx_start: torch.Tensor, block_tables: torch.Tensor,
               max_q_len: int, block_size: int,
               max_blocks: int | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Where the nodes of drafted trees go and what they see: ``(positions, slot_mapping, mask)``.

    Node i of sequence s is packed row ``cu_q[s] + i`` (int32 ``[S + 1]``); ``parents`` (int32 ``[N]``) holds
    each node's parent by its number in the tree, which is below the node's own (anything else: a
    root). ``positions`` (int64 ``[N]``) are ``ctx_start[s]`` + depth; ``slot_mapping`` (int64 ``[N]``) the
    pool slots of cache indexes ``ctx_start[s] + i`` (-1 past the table); ``mask`` (int64 ``[N, W]``,
    ``W = ceil(max_q_len / 64)``) has bit ``j % 64`` of word ``j // 64`` set for the nodes j on the path to the
    root, the node itself among them: what :func:`paged_tree` takes. Trees of up to 1024 nodes. Rows of no node (a
    padded batch's, and a tree's from ``max_q_len`` on) have position 0, slot -1 and no bits.
    """
    s, mb = _tree_rows(cu_q, block_tables, ctx_start, max_q_len, max_blocks)
    if parents.dtype != _I32 or parents.dim() != 1 or not parents.is_contiguous():
        raise ValueError("parents must be contiguous int32 [N]")
    device = _one_device(parents, cu_q, ctx_start, block_tables)
    n, words = parents.shape[0], (max_q_len + 63) // 64
    positions = parents.new_empty(n, dtype=torch.int64)
    slots, mask = torch.empty_like(positions), positions.new_empty(n, words)
    if n:
        _call_on(device, _native.load().mip_tree_index,
                 (positions.data_ptr(), slots.data_ptr(), mask.data_ptr(), words, parents.data_ptr(), n, cu_q.data_ptr(),
                  ctx_start.data_ptr(), block_tables.data_ptr(), block_tables.stride(0), s, max_q_len, block_size, mb),
                 "mip_tree_index")
    return positions, slots, mask


def _tree_args(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
               cu_q: torch.Tensor, ctx_start: torch.Tensor, mask: torch.Tensor, max_q_len: int, scale: float | None,
               out: torch.Tensor | None, max_blocks: int | None,
               workspace: torch.Tensor | None) -> tuple[tuple | None, torch.Tensor, torch.Tensor | None]:
    """Validate a :func:`paged_tree` call: the arguments of ``mip_paged_tree`` up to the stream (None for a call that
    has nothing to do), the output and the scratch memory."""
    rows, pool, strides = q.shape, k_cache.shape, q.stride()
    if len(rows) != 3 or strides[2] != 1:
        raise ValueError("q must be [N, Hq, D] with a contiguous last dimension")
    if len(pool) != 4 or pool != v_cache.shape or not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("k_cache/v_cache must be contiguous [num_blocks, Hkv, block_size, D] tensors of one shape")
    nb, hkv, bs, d = pool
    n, hq, dq = rows
    if dq != d or hkv == 0 or hq == 0 or hq % hkv:
        raise ValueError(f"q {tuple(rows)} does not match the pool (Hkv={hkv}, D={d})")
    dtype = q.dtype
    if not dtype == k_cache.dtype == v_cache.dtype:
        raise TypeError("q and the cache must share one dtype")
    s, mb = _tree_rows(cu_q, block_tables, ctx_start, max_q_len, max_blocks)
    words, bits, bit_strides = (max_q_len + 63) // 64, mask.shape, mask.stride()
    if mask.dtype != torch.int64 or len(bits) != 2 or bits[0] != n or bits[1] < words or (
            bits[1] > 1 and bit_strides[1] != 1):
        raise ValueError(f"mask must be int64 [{n}, >= {words}] with contiguous rows, got {tuple(bits)} {mask.dtype}")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 2.0**-149 <= scale <= 2.0**127:  # in base 2 it has to be an fp32 number
        raise ValueError(f"scale={scale} must be positive and at most 2^127")
    if out is None:
        device = _one_device(q, k_cache, v_cache, block_tables, cu_q, ctx_start, mask)
        out, to = torch.empty_like(q, memory_format=torch.contiguous_format), (hq * d, d)
    else:
        to = out.stride()
        if out.shape != rows or out.dtype != dtype or to[2] != 1:
            raise ValueError("out must be [N, Hq, D] in q's dtype with a contiguous last dimension")
        device = _one_device(q, k_cache, v_cache, block_tables, cu_q, ctx_start, mask, out)
    if not (n and s and max_q_len):
        return None, out, None
    code = dtype_code(dtype)
    workspace = _scratch(workspace, device, _tree_bytes(device, s, max_q_len, hq, hkv, d, bs, mb, code))
    ws_ptr, ws_bytes = _extent(workspace)
    return (out.data_ptr(), to[0], to[1], q.data_ptr(), strides[0], strides[1], k_cache.data_ptr(),
            v_cache.data_ptr(), nb, block_tables.data_ptr(), block_tables.stride(0), cu_q.data_ptr(),
            ctx_start.data_ptr(), mask.data_ptr(), max(bit_strides[0], bits[1]) if n == 1 else bit_strides[0],
            bits[1], s, max_q_len, hq, hkv, d, bs, mb, scale, ws_ptr, ws_bytes, code), out, workspace


def paged_tree(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
               cu_q: torch.Tensor, ctx_start: torch.Tensor, mask: torch.Tensor, max_q_len: int,
               scale: float | None = None, out: torch.Tensor | None = None, max_blocks: int | None = None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of drafted trees' nodes over their sequences' paged keys and each other.

    ``q``: ``[N, Hq, D]`` packed rows (last dim contiguous); sequence ``s`` owns rows ``cu_q[s] ..
    cu_q[s + 1] - 1`` (int32 ``[S + 1]``), whose keys and values are in the pool at cache indexes
    ``ctx_start[s] + i`` (int32 ``[S]``; append them first). A row sees its sequence's ``ctx_start[s]`` cached keys and
    the nodes that its bits in ``mask`` (int64 ``[N, W]``, ``W >= ceil(max_q_len / 64)``, rows contiguous) name; a row that sees
    nothing becomes zeros, and what a row does not see has no influence on it. Returns ``out [N, Hq, D]``; rows of no
    sequence are not written. No reference counterpart (one token a step there, engine/kv_cache.py:615-620).

    16-bit types at head_dim 64 / 128 run on the matrix cores, long contexts of few rows cut into pieces and
    combined; fp32 at those head sizes on the fp32 matrix cores; other head sizes (powers of two from 8 to 256) and short
    calls one query row at a time. Scratch memory is allocated for the call on the current stream, unless ``workspace``
    (:func:`tree_workspace_bytes`) is given, which calls that may run at once must not share. ``out`` must not overlap
    the inputs.
    """
    args, out, workspace = _tree_args(q, k_cache, v_cache, block_tables, cu_q, ctx_start, mask, max_q_len, scale, out,
                                      max_blocks, workspace)
    if args is not None:
        _call_on(q.device, _native.load().mip_paged_tree, args, "mip_paged_tree")
    return out


class TreeStepCalls(PrefillStepCalls):
    """The layer calls of one step of drafted trees; the nodes are appended as a packed prefill's tokens are.

    Each call has scratch memory of its own, as :func:`paged_tree`'s do: layers may run on any stream, and in several
    graphs."""

    def __init__(self, block_tables: torch.Tensor, cu_q: torch.Tensor, ctx_start: torch.Tensor, mask: torch.Tensor,
                 slot_mapping: torch.Tensor, max_q_len: int, scale: float) -> None:
        super().__init__(block_tables, cu_q, ctx_start, slot_mapping, max_q_len, scale)
        self.mask = mask

    def attend(self, layer: int, q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor) -> torch.Tensor:
        """:func:`paged_tree` of one layer; returns ``[1, Hq, N, D]``, a view of ``[N, Hq, D]``."""
        key = (_layout(q), _layout(k_pool), _layout(v_pool))
        hit = self._hit("attend", key, layer)
        if hit is not None:
            _, at, _, kb, vb, step, _ = hit
            _, hq, n, d = q.shape
            out = torch.empty_strided((1, hq, n, d), (hq * d, d, hq * d, 1), dtype=q.dtype, device=q.device)
            if step.workspace_bytes:
                # A copy of the struct, as another thread may be at a call of this step.
                workspace = _scratch(None, q.device, step.workspace_bytes)
                step = _native.TreeStep.from_buffer_copy(step)
                step.workspace, at = workspace.data_ptr(), ctypes.addressof(step)
            _call_on(q.device, _native.load().mip_tree_step_attend,
                     (at, out.data_ptr(), q.data_ptr(), k_pool.data_ptr() + layer * kb, v_pool.data_ptr() + layer * vb),
                     "mip_tree_step_attend")
            return out
        q1 = q[0].transpose(0, 1)
        a, out, workspace = _tree_args(q1, k_pool[layer], v_pool[layer], self.block_tables, self.cu_q, self.ctx_start,
                                       self.mask, self.max_q_len, self.scale, None, None, None)
        if a is not None:
            _call_on(q.device, _native.load().mip_paged_tree, a, "mip_paged_tree")
            if q.shape[0] == 1:
                step = _native.TreeStep(a[1], a[2], a[4], a[5], a[8], a[9], a[10], a[11], a[12], a[13], a[14], None, a[25],
                                        *a[15:23], a[26], a[23])
                self._keep("attend", key, step, k_pool, v_pool, (self.block_tables, self.cu_q, self.ctx_start, self.mask))
        return out.transpose(0, 1).unsqueeze(0)


def tree_workspace_bytes(num_seqs: int, max_q_len: int, num_heads: int, num_kv_heads: int, head_dim: int,
                         block_size: int, max_blocks: int, dtype: torch.dtype) -> int:
    """Bytes of scratch a :func:`paged_tree` call of this shape needs on the current device
    (``mip_paged_tree_workspace``)."""
    return int(_native.load().mip_paged_tree_workspace(num_seqs, max_q_len, num_heads, num_kv_heads, head_dim,
                                                       block_size, max_blocks, dtype_code(dtype)))


def tree_verify(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, cu_q: torch.Tensor, max_q_len: int,
                workspace: torch.Tensor | None = None
                ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Greedy verification of drafted trees: ``(target, path, counts, next_token)``.

    ``logits`` ``[N, vocab]`` (rows contiguous): the model's answer after every node; ``tokens`` int64 ``[N]`` the
    nodes' tokens, ``parents`` and ``cu_q`` as for :func:`tree_index`. ``target`` (int64 ``[N]``): the lowest index
    of each row's greatest logit (a NaN counts as the greatest). ``path`` (int32 ``[S, max_q_len]``, -1 past the
    end) starts at node 0 and goes on to the lowest child whose token is the last node's target, until there is none (of
    siblings that carry one token the first, whatever follows the others);
    ``counts`` (int32 ``[S]``) are the paths' lengths and ``next_token`` (int64 ``[S]``) the target of each one's last node
    (an empty tree: 0 and -1). Scratch memory as for :func:`paged_tree`.
    """
    rows, strides, seqs = logits.shape, logits.stride(), cu_q.shape
    if len(rows) != 2 or rows[1] < 1 or (rows[1] > 1 and strides[1] != 1):
        raise ValueError("logits must be [N, vocab] with contiguous rows")
    n, vocab = rows
    code = dtype_code(logits.dtype)
    if tokens.dtype != torch.int64 or tokens.shape != rows[:1] or not tokens.is_contiguous():
        raise ValueError(f"tokens must be contiguous int64 [{n}]")
    if parents.dtype != _I32 or parents.shape != rows[:1] or not parents.is_contiguous():
        raise ValueError(f"parents must be contiguous int32 [{n}]")
    if cu_q.dtype != _I32 or len(seqs) != 1 or seqs[0] < 1 or not cu_q.is_contiguous():
        raise ValueError("cu_q must be contiguous int32 [S + 1]")
    if max_q_len < 0:
        raise ValueError(f"max_q_len={max_q_len} is negative")
    s, row_stride = seqs[0] - 1, max(strides[0], vocab) if n <= 1 else strides[0]
    if row_stride < vocab:
        raise ValueError("the rows of logits overlap")
    device = _one_device(logits, tokens, parents, cu_q)
    target, following = torch.empty_like(tokens), tokens.new_empty(s)
    path, counts = cu_q.new_empty(s, max_q_len), cu_q.new_empty(s)
    if n or s:
        lib = _native.load()
        workspace = _scratch(workspace, device, _verify_bytes(n, vocab, code))
        ws_ptr, ws_bytes = _extent(workspace)
        _call_on(device, lib.mip_tree_verify,
                 (target.data_ptr(), path.data_ptr(), counts.data_ptr(), following.data_ptr(), logits.data_ptr(),
                  row_stride, n, vocab, tokens.data_ptr(), parents.data_ptr(), cu_q.data_ptr(), s, max_q_len, ws_ptr,
                  ws_bytes, code), "mip_tree_verify")
    return target, path, counts, following


def tree_commit(k_pool: torch.Tensor, v_pool: torch.Tensor, block_tables: torch.Tensor, ctx_start: torch.Tensor,
                path: torch.Tensor, counts: torch.Tensor, max_blocks: int | None = None) -> None:
    """Move the accepted nodes' keys and values to the places of consecutive tokens, every layer, in place.

    ``k_pool``/``v_pool``: ``[num_layers, num_blocks + 1, Hkv, block_size, D]`` contiguous. ``path`` (int32 ``[S, P]``) and
    ``counts`` (int32 ``[S]``) as :func:`tree_verify` returns them: the row of cache index ``ctx_start[s] + path[s, d]``
    moves to ``ctx_start[s] + d`` for ``d < counts[s]``, as if all were read before any is written. A path rises and
    has ``path[s, d] >= d``; an entry that breaks this, or whose place lies outside the table or the pool, ends it.
    No two sequences may own the blocks that rows move in (a block that a fork shares is copied before the nodes are
    appended: ``PagedKVCache.prepare_writes``).
    """
    pool, dtype = k_pool.shape, k_pool.dtype
    if len(pool) != 5 or pool != v_pool.shape or not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError("k_pool/v_pool must be contiguous [L, num_blocks, Hkv, block_size, D] tensors of one shape")
    if dtype != v_pool.dtype:
        raise TypeError("the pools must share one dtype")
    if not path.dtype == counts.dtype == ctx_start.dtype == block_tables.dtype == _I32:
        raise TypeError("path, counts, ctx_start and block_tables must be int32")
    seqs, steps, tab, step, row = counts.shape, path.shape, block_tables.shape, path.stride(), block_tables.stride()
    if len(seqs) != 1 or ctx_start.shape != seqs or len(steps) != 2 or steps[0] != seqs[0]:
        raise ValueError("path must be int32 [S, P], counts and ctx_start int32 [S]")
    s, most = steps
    if len(tab) != 2 or tab[0] < s or tab[1] < 1 or row[1] != 1:
        raise ValueError("block_tables must be int32 [S, max_blocks] with contiguous rows")
    if not (counts.is_contiguous() and ctx_start.is_contiguous()) or (most > 1 and step[1] != 1) or (
            s > 1 and step[0] < most):
        raise ValueError("counts, ctx_start and the rows of path must be contiguous")
    mb = tab[1] if max_blocks is None else int(max_blocks)
    if mb < 1 or mb > tab[1]:
        raise ValueError(f"max_blocks={mb} is outside [1, {tab[1]}]")
    layers, nb, hkv, bs, d = pool
    code = dtype_code(dtype)
    device = _one_device(k_pool, v_pool, block_tables, ctx_start, path, counts)
    if s == 0 or most == 0:
        return
    _call_on(device, _native.load().mip_tree_commit,
             (k_pool.data_ptr(), v_pool.data_ptr(), layers, nb, hkv, d, bs, block_tables.data_ptr(),
              row[0], mb, ctx_start.data_ptr(), path.data_ptr(), max(step[0], most), most, counts.data_ptr(), s, code),
             "mip_tree_commit")
