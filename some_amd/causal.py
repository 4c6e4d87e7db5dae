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
    shape = x.shape
    if len(shape) != 3 or shape[1] == 0 or (head_dim and shape[2] != head_dim):
        raise ValueError(f'{name} must be [rows, heads, head_dim{"" if not head_dim else f" = {head_dim}"}], got {tuple(shape)}')
    if shape[2] not in HEAD_DIMS:
        raise ValueError(f'{name}: head_dim must be one of {HEAD_DIMS}, got {shape[2]}')
    return x


def readable(x: torch.Tensor) -> torch.Tensor:
    """``x`` itself if the library reads its layout in place, else a contiguous copy."""
    return x if _place(x) is not None else aligned(x)


def aligned(x: torch.Tensor) -> torch.Tensor:
    x = x.contiguous()
    return x.clone() if x.data_ptr() & 15 else x


def _place(x: torch.Tensor):
    """(address, row stride, head stride) of a [.., rows, heads, head_dim] tensor, None if the library cannot read it in place.  A dimension of
    one entry has no stride to speak of."""
    p, st, shape = x.data_ptr(), x.stride(), x.shape
    if shape[-3] == 0:
        return 0, 0, 0
    row, head = st[-3] if shape[-3] > 1 else 0, st[-2] if shape[-2] > 1 else 0
    mask = 3 if x.dtype is torch.float32 else 7                     # 16 bytes in elements
    if p & 15 or st[-1] != 1 or row < 0 or head < 0 or (row | head) & mask or row >= _MAX_ROW_BYTES // x.element_size():
        return None
    return p, row, head


def check_device(device: torch.device, *tensors):
    first, want = tensors[0].get_device(), device.index            # (get_device: -1 on the host; a torch.device per tensor is 2 us of a 12 us call)
    for t in tensors:
        i = t.get_device()
        if i != first or i < 0 or (want is not None and i != want):
            raise ValueError(f'a tensor is on {t.device}: the operators run on {device}, all tensors of a call on one device')


_get_device, _raw_stream = torch._C._cuda_getDevice if hasattr(torch._C, '_cuda_getDevice') else torch.cuda.current_device, getattr(torch._C, '_cuda_getCurrentRawStream', None)


def stream_of(t: torch.Tensor) -> int:
    """Address of the current stream of the tensor's device (torch.cuda.current_stream builds an object per call: 3 us of a 10 us call)."""
    return _raw_stream(t.device.index) if _raw_stream is not None else torch.cuda.current_stream(t.device).cuda_stream


class on_device:
    """Makes the tensors' device current around a launch (a stream belongs to its device)."""
    __slots__ = ('want', 'prev')

    def __init__(self, t: torch.Tensor):
        self.want, self.prev = t.device.index, _get_device()

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
    check_device(device, q, k, gamma_q, gamma_k, positions)
    return q, k


def _gain(g: torch.Tensor) -> torch.Tensor:
    return g if g.is_contiguous() and not g.data_ptr() & 15 else aligned(g)


def norm_rope_forward(lib, h, stream, q, k, gamma_q, gamma_k, positions, theta, eps):
    """Launch on checked [rows, heads, head_dim] views -> two new contiguous tensors."""
    q, k, gamma_q, gamma_k, positions = readable(q), readable(k), _gain(gamma_q), _gain(gamma_k), positions.contiguous()
    (M, H, D), G = q.shape, k.shape[1]
    yq, yk = q.new_empty((M, H, D)), k.new_empty((M, G, D))
    rc = lib.some_op_qk_norm_rope(h, DTYPES[q.dtype], D, *_place(q), H, *_place(k), G, M, gamma_q.data_ptr(), gamma_k.data_ptr(), positions.data_ptr(),
                                  positions.dtype is torch.int64, theta, eps, yq.data_ptr(), H * D, D, yk.data_ptr(), G * D, D, stream)
    if rc:
        _lib.check(h, rc)
    return yq, yk


def norm_rope_backward(lib, h, stream, q, k, gamma_q, gamma_k, positions, theta, eps, dyq, dyk, dgq, dgk, accumulate):
    """-> (dq, dk); the gain gradients go into ``dgq`` / ``dgk``."""
    q, k, gamma_q, gamma_k, positions = readable(q), readable(k), _gain(gamma_q), _gain(gamma_k), positions.contiguous()
    dyq, dyk = readable(dyq), readable(dyk)
    (M, H, D), G = q.shape, k.shape[1]
    dq, dk = q.new_empty((M, H, D)), k.new_empty((M, G, D))
    n = lib.some_train_qk_norm_rope_bytes(h, M, H, G, D)
    work = gamma_q.new_empty((n + 3) // 4)
    rc = lib.some_train_qk_norm_rope_bwd(h, DTYPES[q.dtype], D, *_place(q), H, *_place(k), G, M, gamma_q.data_ptr(), gamma_k.data_ptr(), positions.data_ptr(),
                                         positions.dtype is torch.int64, theta, eps, *_place(dyq), *_place(dyk), dq.data_ptr(), H * D, D, dk.data_ptr(),
                                         G * D, D, dgq.data_ptr(), dgk.data_ptr(), accumulate, work.data_ptr(), n, stream)
    if rc:
        _lib.check(h, rc)
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
    check_device(device, q, k, v, batch.frame_offsets_dev, kv.frame_offsets_dev)
    return q, k, v, kv


def attention_forward(lib, h, stream, q, k, v, batch, kv, causal, scale, for_backward):
    """Launch on checked, readable views -> (out, rest, lse), the last two None unless ``for_backward`` (rest: 16-bit types alone)."""
    (M, H, D), (N, G, _) = q.shape, k.shape
    out = q.new_empty((M, H, D))
    lse = torch.empty((H, M), dtype=torch.float32, device=q.device) if for_backward else None
    rest = torch.empty_like(out) if for_backward and q.dtype is not torch.float32 else None
    n = lib.some_op_causal_attention_bytes(h, DTYPES[q.dtype], H, G, D, batch.B, M, N)
    work = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    rc = lib.some_op_causal_attention(h, DTYPES[q.dtype], D, *_place(q), H, *_place(k), *_place(v), G, batch.frame_offsets_dev.data_ptr(),
                                      kv.frame_offsets_dev.data_ptr(), batch.B, M, N, causal, scale, out.data_ptr(), H * D, D,
                                      rest.data_ptr() if rest is not None else None, lse.data_ptr() if for_backward else None, work.data_ptr() if n else None, n, stream)
    if rc:
        _lib.check(h, rc)
    return out, rest, lse


def attention_backward(lib, h, stream, q, k, v, batch, kv, causal, scale, out, rest, lse, dout):
    dout = readable(dout)
    (M, H, D), (N, G, _) = q.shape, k.shape
    dq, dk, dv = q.new_empty((M, H, D)), k.new_empty((N, G, D)), v.new_empty((N, G, D))
    n = lib.some_train_causal_attention_bytes(h, DTYPES[q.dtype], H, G, D, batch.B, M, N)
    work = torch.empty(n, dtype=torch.uint8, device=q.device)
    rc = lib.some_train_causal_attention_bwd(h, DTYPES[q.dtype], D, *_place(q), H, *_place(k), *_place(v), G, batch.frame_offsets_dev.data_ptr(),
                                             kv.frame_offsets_dev.data_ptr(), batch.B, M, N, causal, scale, out.data_ptr(), H * D, D,
                                             rest.data_ptr() if rest is not None else None, lse.data_ptr(),
                                             *_place(dout), dq.data_ptr(), H * D, D, dk.data_ptr(), G * D, D, dv.data_ptr(), G * D, D, work.data_ptr(), n,
                                             stream)
    if rc:
        _lib.check(h, rc)
    return dq, dk, dv


def check_step(device, q, k_cache, v_cache, lengths, max_length):
    """-> (q, the caches' places, max_length), checked."""
    q = heads_view(q, 'q', 0)
    B, H, D = q.shape
    shape = k_cache.shape if isinstance(k_cache, torch.Tensor) else ()
    for name, c in (('k_cache', k_cache), ('v_cache', v_cache)):
        if not isinstance(c, torch.Tensor) or c.shape != shape or len(shape) != 4 or shape[0] != B or shape[2] == 0 or shape[3] != D:
            raise ValueError(f'{name} must be [{B}, capacity, kv_heads, {D}], k and v alike')
        if c.dtype is not q.dtype:
            raise TypeError(f'q and {name} must have one type, got {q.dtype} and {c.dtype}')
    _, capacity, G, _ = shape
    if H % G:
        raise ValueError(f'{H} query heads are not a multiple of {G} key / value heads')
    if not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or lengths.shape != (B,):
        raise ValueError(f'lengths must be int32 [{B}]')
    max_length = capacity if max_length is None else int(max_length)
    if not 0 <= max_length <= capacity:
        raise ValueError(f'max_length {max_length} outside the cache of {capacity} frames')
    check_device(device, q, k_cache, v_cache, lengths)
    places = []
    for name, c in (('k_cache', k_cache), ('v_cache', v_cache)):
        p, stride = _place(c), c.stride(0) if B > 1 else 0
        if p is None or stride < 0 or stride & (3 if c.dtype is torch.float32 else 7):
            raise ValueError(f'{name}: unsupported layout (head_dim contiguous, 16-byte aligned rows, heads and streams; a copy per frame is refused)')
        places += [p[0], stride, p[1], p[2]]
    return q, places, max_length


def attention_step(lib, h, stream, q, places, G, lengths, max_length, scale):
    q, lengths = readable(q), lengths.contiguous()
    B, H, D = q.shape
    out = q.new_empty((B, H, D))
    n = lib.some_op_attention_step_bytes(h, DTYPES[q.dtype], B, H, G, D, max_length)
    work = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    rc = lib.some_op_attention_step(h, DTYPES[q.dtype], D, *_place(q), H, *places, G, lengths.data_ptr(), B, max_length, scale, out.data_ptr(), H * D, D,
                                    work.data_ptr() if n else None, n, stream)
    if rc:
        _lib.check(h, rc)
    return out


def no_gradient_lost(what: str, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                break
        else:
            return
        raise RuntimeError(f'{what} is not differentiable: use the operator of the same name in TrainOps, or torch.no_grad()')
