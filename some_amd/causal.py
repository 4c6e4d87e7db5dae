"""Host side of the causal attention operators over packed clips (include/some_amd.h, "causal attention over packed clips"): argument checks,
layouts and launches shared by the serving entry points (``Engine.qk_norm_rope`` / ``causal_attention`` / ``attention_step``) and the differentiable
ones (``TrainOps.qk_norm_rope`` / ``causal_attention``).

Tensors are [rows, heads, head_dim] (or [rows, heads * head_dim], as a linear layer writes them) in float32, float16 or bfloat16, head_dim 64 or 128; any
row and head strides the library takes (slices of a fused projection) are read in place, other layouts are copied first."""
import math

import numpy as np
import torch

from . import _lib

DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
HEAD_DIMS = (64, 128)
_MAX_ROW_BYTES = 1 << 24


def frame_positions(batch) -> torch.Tensor:
    """int32 [total_frames]: every packed frame's index in its clip (cached on the batch descriptor)."""
    cached = getattr(batch, '_positions_dev', None)
    if cached is None:
        n = np.asarray(batch.frame_counts, dtype=np.int64)
        pos = np.arange(batch.total_frames, dtype=np.int64) - np.repeat(np.asarray(batch.frame_offsets[:-1], dtype=np.int64), n)
        cached = batch._positions_dev = torch.from_numpy(pos.astype(np.int32)).to(batch.frame_offsets_dev.device)
    return cached


def heads_view(x: torch.Tensor, name: str, head_dim: int) -> torch.Tensor:
    """[rows, heads, head_dim] view of ``x``, checked."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f'{name} must be a tensor')
    if x.dtype not in DTYPES:
        raise TypeError(f'{name} must be float32, float16 or bfloat16, got {x.dtype}')
    if x.dim() == 2:
        if not head_dim:
            raise ValueError(f'{name} is [rows, heads * head_dim]: pass head_dim')
        if x.shape[1] == 0 or x.shape[1] % head_dim:
            raise ValueError(f'{name}: {x.shape[1]} columns are not a multiple of head_dim {head_dim}')
        x = x.unflatten(1, (x.shape[1] // head_dim, head_dim))
    if x.dim() != 3 or x.shape[1] == 0 or (head_dim and x.shape[2] != head_dim):
        raise ValueError(f'{name} must be [rows, heads, head_dim{"" if not head_dim else f" = {head_dim}"}], got {tuple(x.shape)}')
    if x.shape[2] not in HEAD_DIMS:
        raise ValueError(f'{name}: head_dim must be one of {HEAD_DIMS}, got {x.shape[2]}')
    return x


def readable(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself if the library reads its layout in place, else a contiguous copy."""
    size = x.element_size()
    if x.stride(-1) == 1 and not x.data_ptr() & 15:
        for n, s in zip(x.shape[:-1], x.stride()[:-1]):
            if n > 1 and (s < 0 or s * size & 15):
                break
        else:
            if x.shape[-3] <= 1 or x.stride(-3) * size < _MAX_ROW_BYTES:
                return x
    x = x.contiguous()
    return x if not x.data_ptr() & 15 else x.clone()


def _rows(x: torch.Tensor):
    """(address, row stride, head stride) of a [..., rows, heads, head_dim] tensor; a dimension of one entry has no stride to speak of."""
    return x.data_ptr(), x.stride(-3) if x.shape[-3] > 1 else 0, x.stride(-2) if x.shape[-2] > 1 else 0


def check_device(device: torch.device, **tensors):
    for name, t in tensors.items():
        d = t.device
        if d.type != 'cuda' or (device.index is not None and d.index != device.index):
            raise ValueError(f'{name} is on {d}, the operators run on {device}')
    ds = {t.device for t in tensors.values()}
    if len(ds) > 1:
        raise ValueError(f'tensors on several devices: {sorted(map(str, ds))}')


class on_device:
    """Makes the tensors' device current around a launch (a stream belongs to its device)."""

    def __init__(self, t: torch.Tensor):
        self.want, self.prev = t.device.index, torch.cuda.current_device()

    def __enter__(self):
        if self.want != self.prev:
            torch.cuda.set_device(self.want)

    def __exit__(self, *exc):
        if self.want != self.prev:
            torch.cuda.set_device(self.prev)
        return False


def check_norm_rope(device, q, k, gamma_q, gamma_k, positions):
    """-> (q, k) as checked [rows, heads, head_dim] views."""
    if not isinstance(gamma_q, torch.Tensor) or gamma_q.dim() != 1:
        raise ValueError('gamma_q must be [head_dim]')
    D = gamma_q.shape[0]
    q, k = heads_view(q, 'q', D), heads_view(k, 'k', D)
    if q.dtype != k.dtype:
        raise TypeError(f'q and k must have one type, got {q.dtype} and {k.dtype}')
    if q.shape[0] != k.shape[0]:
        raise ValueError(f'q has {q.shape[0]} rows, k {k.shape[0]}')
    for name, g in (('gamma_q', gamma_q), ('gamma_k', gamma_k)):
        if not isinstance(g, torch.Tensor) or g.dtype != torch.float32 or g.shape != (D,):
            raise ValueError(f'{name} must be float32 [{D}]')
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape != (q.shape[0],):
        raise ValueError(f'positions must be int32 or int64 [{q.shape[0]}], got {positions.dtype} {tuple(positions.shape)}')
    check_device(device, q=q, k=k, gamma_q=gamma_q, gamma_k=gamma_k, positions=positions)
    return q, k


def aligned(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    return x.clone() if x.data_ptr() & 15 else x


def norm_rope_forward(lib, h, stream, q, k, gamma_q, gamma_k, positions, theta, eps):
    """Launch on checked [rows, heads, head_dim] views -> two new contiguous tensors."""
    q, k, gamma_q, gamma_k, positions = readable(q), readable(k), aligned(gamma_q), aligned(gamma_k), positions.contiguous()
    D = q.shape[2]
    yq, yk = q.new_empty(q.shape), k.new_empty(k.shape)
    _lib.check(h, lib.some_op_qk_norm_rope(h, DTYPES[q.dtype], D, *_rows(q), q.shape[1], *_rows(k), k.shape[1], q.shape[0], gamma_q.data_ptr(),
                                           gamma_k.data_ptr(), positions.data_ptr(), positions.dtype == torch.int64, float(theta), float(eps), *_rows(yq),
                                           *_rows(yk), stream))
    return yq, yk


def norm_rope_backward(lib, h, stream, q, k, gamma_q, gamma_k, positions, theta, eps, dyq, dyk, dgq, dgk, accumulate):
    """-> (dq, dk); the gain gradients go into ``dgq`` / ``dgk``."""
    q, k, gamma_q, gamma_k, positions = readable(q), readable(k), aligned(gamma_q), aligned(gamma_k), positions.contiguous()
    dyq, dyk = readable(dyq), readable(dyk)
    D = q.shape[2]
    dq, dk = q.new_empty(q.shape), k.new_empty(k.shape)
    work = torch.empty(lib.some_train_qk_norm_rope_bytes(h, q.shape[0], q.shape[1], k.shape[1], D), dtype=torch.uint8, device=q.device)
    _lib.check(h, lib.some_train_qk_norm_rope_bwd(h, DTYPES[q.dtype], D, *_rows(q), q.shape[1], *_rows(k), k.shape[1], q.shape[0], gamma_q.data_ptr(),
                                                  gamma_k.data_ptr(), positions.data_ptr(), positions.dtype == torch.int64, float(theta), float(eps),
                                                  *_rows(dyq), *_rows(dyk), *_rows(dq), *_rows(dk), dgq.data_ptr(), dgk.data_ptr(), int(accumulate),
                                                  work.data_ptr(), work.numel(), stream))
    return dq, dk


def default_scale(scale, head_dim: int) -> float:
    scale = head_dim ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f'scale must be finite and positive, got {scale}')
    return scale


def check_attention(device, q, k, v, batch, kv_batch, head_dim):
    """-> (q, k, v) as checked views, and the key batch."""
    q = heads_view(q, 'q', head_dim)
    D = q.shape[2]
    k, v = heads_view(k, 'k', D), heads_view(v, 'v', D)
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f'q, k and v must have one type, got {q.dtype}, {k.dtype}, {v.dtype}')
    if k.shape != v.shape:
        raise ValueError(f'k is {tuple(k.shape)}, v {tuple(v.shape)}')
    if q.shape[1] % k.shape[1]:
        raise ValueError(f'{q.shape[1]} query heads are not a multiple of {k.shape[1]} key / value heads')
    kv = batch if kv_batch is None else kv_batch
    if kv.B != batch.B:
        raise ValueError(f'{batch.B} clips of queries, {kv.B} of keys')
    if q.shape[0] != batch.total_frames or k.shape[0] != kv.total_frames:
        raise ValueError(f'q has {q.shape[0]} rows (the batch {batch.total_frames}), k and v {k.shape[0]} (the batch {kv.total_frames})')
    check_device(device, q=q, k=k, v=v, frame_offsets=batch.frame_offsets_dev, kv_frame_offsets=kv.frame_offsets_dev)
    return q, k, v, kv


def attention_forward(lib, h, stream, q, k, v, batch, kv, causal, scale, want_lse):
    """Launch on checked, readable views -> (out, lse or None)."""
    out = q.new_empty(q.shape)
    lse = torch.empty((q.shape[1], q.shape[0]), dtype=torch.float32, device=q.device) if want_lse else None
    n = lib.some_op_causal_attention_bytes(h, q.shape[1], k.shape[1], q.shape[2], batch.B, q.shape[0], k.shape[0])
    work = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    _lib.check(h, lib.some_op_causal_attention(h, DTYPES[q.dtype], q.shape[2], *_rows(q), q.shape[1], *_rows(k), *_rows(v), k.shape[1],
                                               batch.frame_offsets_dev.data_ptr(), kv.frame_offsets_dev.data_ptr(), batch.B, q.shape[0], k.shape[0],
                                               int(causal), scale, *_rows(out), lse.data_ptr() if want_lse else None, work.data_ptr() if n else None, n, stream))
    return out, lse


def attention_backward(lib, h, stream, q, k, v, batch, kv, causal, scale, out, lse, dout):
    dout = readable(dout)
    dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)
    work = torch.empty(lib.some_train_causal_attention_bytes(h, q.shape[1], k.shape[1], q.shape[2], batch.B, q.shape[0], k.shape[0]), dtype=torch.uint8, device=q.device)
    _lib.check(h, lib.some_train_causal_attention_bwd(h, DTYPES[q.dtype], q.shape[2], *_rows(q), q.shape[1], *_rows(k), *_rows(v), k.shape[1],
                                                      batch.frame_offsets_dev.data_ptr(), kv.frame_offsets_dev.data_ptr(), batch.B, q.shape[0], k.shape[0],
                                                      int(causal), scale, *_rows(out), lse.data_ptr(), *_rows(dout), *_rows(dq), *_rows(dk), *_rows(dv),
                                                      work.data_ptr(), work.numel(), stream))
    return dq, dk, dv


def attention_step(lib, h, stream, device, q, k_cache, v_cache, lengths, max_length, scale):
    q = heads_view(q, 'q', 0)
    B, H, D = q.shape
    for name, c in (('k_cache', k_cache), ('v_cache', v_cache)):
        if not isinstance(c, torch.Tensor) or c.dim() != 4 or c.shape[0] != B or c.shape[3] != D or c.shape != k_cache.shape or c.shape[2] == 0:
            raise ValueError(f'{name} must be [{B}, capacity, kv_heads, {D}], k and v alike')
        if c.dtype != q.dtype:
            raise TypeError(f'q and {name} must have one type, got {q.dtype} and {c.dtype}')
    if H % k_cache.shape[2]:
        raise ValueError(f'{H} query heads are not a multiple of {k_cache.shape[2]} key / value heads')
    if not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or lengths.shape != (B,):
        raise ValueError(f'lengths must be int32 [{B}]')
    capacity = k_cache.shape[1]
    max_length = capacity if max_length is None else int(max_length)
    if not 0 <= max_length <= capacity:
        raise ValueError(f'max_length {max_length} outside the cache of {capacity} frames')
    check_device(device, q=q, k_cache=k_cache, v_cache=v_cache, lengths=lengths)
    for name, c in (('k_cache', k_cache), ('v_cache', v_cache)):
        if readable(c) is not c or (B > 1 and (c.stride(0) < 0 or c.stride(0) * c.element_size() & 15)):
            raise ValueError(f'{name}: unsupported layout (head_dim contiguous, 16-byte aligned rows, heads and streams; a copy per frame is refused)')
    scale = default_scale(scale, D)
    q, lengths = readable(q), lengths.contiguous()
    out = q.new_empty(q.shape)
    G = k_cache.shape[2]
    with on_device(q):
        n = lib.some_op_attention_step_bytes(h, B, H, G, D, max_length)
        work = torch.empty(n, dtype=torch.uint8, device=q.device)
        (ka, kr, kh), (va, vr, vh) = _rows(k_cache), _rows(v_cache)
        kb, vb = (k_cache.stride(0), v_cache.stride(0)) if B > 1 else (0, 0)
        _lib.check(h, lib.some_op_attention_step(h, DTYPES[q.dtype], D, *_rows(q), H, ka, kb, kr, kh, va, vb, vr, vh, G, lengths.data_ptr(), B, max_length,
                                                 scale, *_rows(out), work.data_ptr(), n, stream()))
    return out


def no_gradient_lost(what: str, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f'{what} is not differentiable: use the operator of the same name in TrainOps, or torch.no_grad()')
