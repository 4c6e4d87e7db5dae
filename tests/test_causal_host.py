"""What the causal attention operators refuse, without a GPU: the Python checks and the C ABI's."""
import ctypes as C

import pytest
import torch

from some_amd import _lib, causal
from some_amd.configs import get_config
from some_amd.engine import ClipBatch, Engine

CUDA = torch.device('cuda')


def _attn(q=(10, 4, 64), k=(10, 2, 64), v=None, lens=(10,), kv=None, head_dim=0, dtype=torch.float32, kdtype=None):
    q, k, v = (torch.zeros(s, dtype=t) for s, t in ((q, dtype), (k, kdtype or dtype), (v or k, dtype)))
    return causal.check_attention(CUDA, q, k, v, ClipBatch(list(lens), 'cpu'), ClipBatch(list(kv), 'cpu') if kv else None, head_dim)


@pytest.mark.parametrize('kw,msg', [
    (dict(q=(10, 3, 64)), 'multiple of 2'), (dict(q=(10, 4, 80), k=(10, 2, 80)), 'head_dim must be one of'), (dict(k=(10, 2, 128)), 'head_dim = 64'),
    (dict(lens=(9,)), 'rows'), (dict(kv=(9,)), 'rows'), (dict(kv=(5, 5)), 'clips'), (dict(v=(10, 1, 64)), 'k is'),
    (dict(q=(10, 256)), 'pass head_dim'), (dict(q=(10, 250), head_dim=64), 'not a multiple of head_dim'), (dict(q=(10, 0, 64)), 'must be'),
    (dict(), 'on cpu')])
def test_attention_refuses(kw, msg):
    with pytest.raises(ValueError, match=msg):
        _attn(**kw)


def test_types_refused():
    with pytest.raises(TypeError, match='float32, float16 or bfloat16'):
        _attn(dtype=torch.float64)
    with pytest.raises(TypeError, match='one type'):
        _attn(kdtype=torch.float16)
    for s in (0.0, -1.0, float('nan'), float('inf')):
        with pytest.raises(ValueError, match='scale'):
            causal.default_scale(s, 64)
    assert causal.default_scale(None, 64) == 0.125


def _norm(q=(10, 4, 64), k=(10, 2, 64), g=64, gk=64, pos=torch.zeros(10, dtype=torch.int64), gt=torch.float32, kt=torch.float32):
    return causal.check_norm_rope(CUDA, torch.zeros(q), torch.zeros(k, dtype=kt), torch.zeros(g, dtype=gt), torch.zeros(gk), pos)


@pytest.mark.parametrize('kw,msg', [
    (dict(k=(9, 2, 64)), 'rows'), (dict(g=80), 'head_dim'), (dict(gk=128), 'gamma_k'), (dict(gt=torch.float16), 'gamma_q'),
    (dict(pos=torch.zeros(9, dtype=torch.int64)), 'positions'), (dict(pos=torch.zeros(10)), 'positions'), (dict(), 'on cpu')])
def test_norm_rope_refuses(kw, msg):
    with pytest.raises(ValueError, match=msg):
        _norm(**kw)
    with pytest.raises(TypeError, match='one type'):
        _norm(kt=torch.float16)


def test_step_refuses():
    def call(q=(2, 4, 64), k=(2, 9, 2, 64), v=None, n=torch.zeros(2, dtype=torch.int32), m=None, t=torch.float32):
        return causal.check_step(CUDA, torch.zeros(q), torch.zeros(k, dtype=t), torch.zeros(v or k, dtype=t), n, m)
    for kw, msg in [(dict(k=(3, 9, 2, 64)), 'k_cache'), (dict(v=(2, 8, 2, 64)), 'v_cache'), (dict(k=(2, 9, 3, 64)), 'multiple of 3'),
                    (dict(n=torch.zeros(2, dtype=torch.int64)), 'int32'), (dict(n=torch.zeros(3, dtype=torch.int32)), 'lengths'),
                    (dict(m=10), 'max_length'), (dict(m=-1), 'max_length'), (dict(k=(2, 9, 2, 128)), 'k_cache'), (dict(), 'on cpu')]:
        with pytest.raises(ValueError, match=msg):
            call(**kw)
    with pytest.raises(TypeError, match='one type'):
        call(t=torch.bfloat16)


def test_host_only_engine_and_gradients_refused():
    eng = Engine(get_config('two_head_model', lay=0), host_only=True)
    with pytest.raises(RuntimeError, match='host-only'):
        eng.causal_attention(torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), ClipBatch([1], 'cpu'))
    with pytest.raises(RuntimeError, match='not differentiable'):
        causal.no_gradient_lost('x', torch.zeros(1, requires_grad=True))
    with torch.no_grad():
        causal.no_gradient_lost('x', torch.zeros(1, requires_grad=True))


def test_layouts_read_in_place_or_copied():
    x = torch.zeros(8, 6, 64)
    for t in (x, x[:, :3], x[::2], x.transpose(0, 1), x[:, :1].expand(8, 4, 64), x[:0], x[:1, 5:]):
        assert causal.readable(t) is t
    odd = torch.zeros(8, 6 * 64 + 1)[:, 1:].unflatten(1, (6, 64))
    for t in (odd, torch.zeros(8, 64, 6).transpose(1, 2), torch.zeros(2, 1 << 22)[:, :64].unsqueeze(1)):
        c = causal.readable(t)
        assert c is not t and c.is_contiguous() and not c.data_ptr() & 15


def test_frame_positions():
    b = ClipBatch([3, 0, 2, 1], 'cpu')
    p = causal.frame_positions(b)
    assert p.dtype == torch.int32 and p.tolist() == [0, 1, 2, 0, 1, 0] and causal.frame_positions(b) is p
    assert causal.frame_positions(ClipBatch([], 'cpu')).shape == (0,)


def test_c_abi_refuses():
    lib = _lib.load()
    eng = Engine(get_config('two_head_model', lay=0), host_only=True)
    h, p = eng.handle, C.c_void_p(4096)                   # never dereferenced: every call below fails validation

    def attn(dtype=2, D=64, q=p, qs=(256, 64), H=4, k=p, ks=(128, 64), G=2, off=p, B=1, M=10, N=10, scale=0.125, out=p, work=0, rest=None):
        return lib.some_op_causal_attention(h, dtype, D, q, *qs, H, k, *ks, k, *ks, G, off, off, B, M, N, 1, scale, out, *qs, rest, None, p if work else None, work, None)

    def bwd(dtype=2, D=64, H=4, G=2, work=p, n=1 << 30, N=10, scale=0.125, ds=(256, 64), rest=p):
        r = (p, 256, 64)
        return lib.some_train_causal_attention_bwd(h, dtype, D, *r, H, *r, *r, G, p, p, 1, 10, N, 1, scale, *r, rest, p, p, *ds, *r, *r, *r, work, n, None)

    def step(dtype=2, D=64, H=4, G=2, B=3, m=2000, work=p, n=1 << 30, kb=128 * 2000, scale=0.125, lengths=p):
        return lib.some_op_attention_step(h, dtype, D, p, 256, 64, H, p, kb, 128, 64, p, kb, 128, 64, G, lengths, B, m, scale, p, 256, 64, work, n, None)

    def rope(dtype=2, D=64, H=4, G=2, rows=10, pos=p, p64=0, theta=1e4, eps=1e-6, g=p):
        r = (p, 256, 64)
        return lib.some_op_qk_norm_rope(h, dtype, D, *r, H, *r, G, rows, g, g, pos, p64, theta, eps, *r, *r, None)

    def rope_bwd(n=1 << 30, D=64, theta=1e4, dg=p):
        r = (p, 256, 64)
        return lib.some_train_qk_norm_rope_bwd(h, 2, D, *r, 4, *r, 2, 10, p, p, p, 0, theta, 1e-6, *r, *r, *r, *r, dg, p, 0, p, n, None)

    odd = C.c_void_p(4104)
    cases = [(attn, dict(dtype=3), b'dtype'), (attn, dict(dtype=-1), b'dtype'), (attn, dict(D=96), b'head_dim'), (attn, dict(H=3), b'multiple'), (attn, dict(G=0), b'multiple'),
             (attn, dict(H=2048, G=2048), b'1024'), (attn, dict(q=odd), b'aligned'), (attn, dict(qs=(260, 64)), b'aligned'), (attn, dict(ks=(-128, 64)), b'aligned'),
             (attn, dict(qs=(1 << 24, 64)), b'16 MiB'), (attn, dict(q=None), b'null'), (attn, dict(off=None), b'null'), (attn, dict(k=None), b'null'),
             (attn, dict(B=-1), b'2^29'), (attn, dict(M=1 << 29), b'2^29'), (attn, dict(scale=0.0), b'scale'), (attn, dict(scale=float('nan')), b'scale'),
             (attn, dict(B=1 << 28, H=1024, G=1), b'one launch'),
             (bwd, dict(dtype=5), b'dtype'), (bwd, dict(H=3), b'multiple'), (bwd, dict(work=None), b'null'), (bwd, dict(work=odd), b'aligned'), (bwd, dict(N=1 << 29), b'2^29'), (bwd, dict(scale=-1.0), b'scale'),
             (bwd, dict(ds=(255, 64)), b'aligned'),
             (step, dict(dtype=3), b'dtype'), (step, dict(H=5), b'multiple'), (step, dict(B=65536), b'65535'), (step, dict(B=65535, H=1024, G=1024, m=1), b'one launch'), (rope, dict(rows=(1 << 29) - 1, H=1024, G=1), b'one launch'), (step, dict(B=-1), b'65535'), (step, dict(m=-1), b'max_length'),
             (step, dict(kb=4), b'aligned'), (step, dict(kb=-128), b'aligned'), (step, dict(lengths=None), b'null'), (step, dict(scale=0.0), b'scale'), (step, dict(work=odd), b'aligned'),
             (rope, dict(D=32), b'head_dim'), (rope, dict(H=0), b'heads'), (rope, dict(rows=-1), b'rows'), (rope, dict(pos=None), b'null'),
             (rope, dict(pos=C.c_void_p(4100), p64=1), b'positions'), (rope, dict(theta=0.0), b'theta'), (rope, dict(theta=float('inf')), b'theta'),
             (rope, dict(eps=-1.0), b'eps'), (rope, dict(g=odd), b'gains'), (rope_bwd, dict(D=32), b'head_dim'), (rope_bwd, dict(theta=-1.0), b'theta'), (rope_bwd, dict(dg=None), b'null')]
    for fn, kw, msg in cases:
        assert fn(**kw) == _lib.SOME_EINVAL, (fn.__name__, kw)
        assert msg in lib.some_last_error(h), (fn.__name__, kw, lib.some_last_error(h))
    assert step(n=16) == _lib.SOME_ENOMEM and b'workspace' in lib.some_last_error(h)
    assert step(work=None) == _lib.SOME_ENOMEM
    assert attn(rest=odd) == bwd(rest=odd) == _lib.SOME_EINVAL and b'rest must be' in lib.some_last_error(h)
    assert bwd(n=16) == _lib.SOME_ENOMEM and b'workspace' in lib.some_last_error(h)
    assert attn(N=100000) == _lib.SOME_ENOMEM and attn(N=100000, work=4096) == _lib.SOME_ENOMEM         # few queries over many keys: cut into parts
    assert lib.some_op_causal_attention_bytes(h, 2, 4, 2, 64, 1, 10, 100000) > 0 == lib.some_op_causal_attention_bytes(h, 2, 8, 8, 64, 32, 82688, 82688)
    assert rope_bwd(n=16) == _lib.SOME_ENOMEM and b'scratch' in lib.some_last_error(h)
    # nothing to do: no launch, no error
    assert attn(M=0) == attn(B=0) == step(B=0) == rope(rows=0) == _lib.SOME_OK
    assert lib.some_op_attention_step_bytes(h, 2, 3, 4, 2, 64, 2000) >= 3 * 4 * 2 * 66 * 4
    for bad in ((0, 4, 2, 64, 10), (1, 3, 2, 64, 10), (1, 4, 0, 64, 10), (1, 4, 2, 64, 0)):
        assert lib.some_op_attention_step_bytes(h, 2, *bad) == 256
    assert lib.some_train_qk_norm_rope_bytes(h, -1, 4, 2, 64) == 256 and lib.some_train_qk_norm_rope_bytes(h, 0, 4, 2, 64) >= 2 * 64 * 4
