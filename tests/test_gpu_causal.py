"""Causal attention over packed clips, the norm + rotation in front of it and the single-frame step on a real MI355X, against 64-bit definitions
with derived bounds (tests/causal_oracle.py)."""
import math

import numpy as np
import pytest
import torch

import causal_oracle as oracle
from some_amd.configs import get_config

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope='module')
def eng():
    from some_amd.engine import Engine
    return Engine(get_config('two_head_model', lay=0), device='cuda')


@pytest.fixture(scope='module')
def ops(eng):
    from some_amd.training.ops import TrainOps
    return TrainOps(eng)


def _batch(lens):
    from some_amd.engine import ClipBatch
    return ClipBatch(lens, 'cuda')


def _normal(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(*shape, device='cuda', generator=g) * scale).to(dtype)


def _qkv(seed, M, N, H, G, D, dtype):
    return _normal(seed, M, H, D, dtype=dtype), _normal(seed + 1, N, G, D, dtype=dtype), _normal(seed + 2, N, G, D, dtype=dtype)


# ---- norm + rotation --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,H,G,D', [(1, 1, 1, 64), (3, 8, 2, 64), (129, 5, 1, 128), (1000, 8, 8, 64), (2049, 12, 4, 128), (257, 33, 3, 64)])
def test_norm_rope(ops, eng, dtype, M, H, G, D):
    q, k = _normal(1, M, H, D, dtype=dtype, scale=3.0), _normal(2, M, G, D, dtype=dtype, scale=0.1)
    gq, gk = 1 + _normal(3, D, scale=0.3), 1 + _normal(4, D, scale=0.3)
    pos = torch.randint(-50, 3000000, (M,), device='cuda', generator=torch.Generator(device='cuda').manual_seed(5))
    if M % 2:
        pos = pos.int()
    dq, dk = _normal(6, M, H, D, dtype=dtype), _normal(7, M, G, D, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, gq, gk)]
    yq, yk = ops.qk_norm_rope(*leaves, pos)
    grads = torch.autograd.grad([yq, yk], leaves, [dq, dk])
    sq, sk = eng.qk_norm_rope(q, k, gq, gk, pos)
    assert torch.equal(sq, yq) and torch.equal(sk, yk)
    for x, g, d, y, dx, dg in ((q, gq, dq, yq, grads[0], grads[2]), (k, gk, dk, yk, grads[1], grads[3])):
        w = oracle.norm_rope(x, g, pos, dy=d)
        oracle.check(y.detach(), *w[0:2], 'y')
        oracle.check(dx, *w[2:4], 'dx')
        oracle.check(dg, *w[4:6], 'dgamma')


def test_norm_rope_views_theta_eps_and_no_rows(ops, eng):
    M, H, G, D = 77, 6, 3, 64
    fused = _normal(11, M, H + 2 * G, D, dtype=torch.bfloat16)
    flat = fused.view(M, -1)
    gq, gk, pos = torch.ones(D, device='cuda'), torch.full((D,), 0.5, device='cuda'), torch.arange(M, device='cuda', dtype=torch.int32)
    a = eng.qk_norm_rope(fused[:, :H], fused[:, H:H + G], gq, gk, pos, theta=500.0, eps=0.25)
    b = eng.qk_norm_rope(flat[:, :H * D], flat[:, H * D:(H + G) * D], gq, gk, pos, theta=500.0, eps=0.25)
    assert b[0].shape == (M, H * D) and torch.equal(a[0].view(M, -1), b[0]) and torch.equal(a[1].view(M, -1), b[1])
    oracle.check(a[0], *oracle.norm_rope(fused[:, :H], gq, pos, theta=500.0, eps=0.25))
    odd = torch.zeros(M, H * D + 3, device='cuda', dtype=torch.bfloat16)[:, 3:].copy_(flat[:, :H * D])       # rows not 16-byte aligned: copied
    c = eng.qk_norm_rope(odd, flat[:, H * D:(H + G) * D], gq, gk, pos, theta=500.0, eps=0.25)
    assert torch.equal(c[0], b[0])
    z = eng.qk_norm_rope(fused[:0, :H], fused[:0, H:H + G], gq, gk, pos[:0])
    assert z[0].shape == (0, H, D) and z[1].shape == (0, G, D)
    leaves = [t.detach().clone().requires_grad_() for t in (fused[:0, :H], fused[:0, H:H + G], gq, gk)]
    y = ops.qk_norm_rope(*leaves, pos[:0])
    (y[0].sum() + y[1].sum()).backward()
    assert not leaves[2].grad.any() and not leaves[3].grad.any()
    zero = torch.zeros(5, 2, D, device='cuda')                                                               # a head of zeros is finite
    assert not eng.qk_norm_rope(zero, zero, gq, gk, pos[:5])[0].any()


def test_norm_rope_gradient_of_one_output_and_differences(ops):
    M, H, G, D = 9, 4, 2, 64
    x, k = _normal(21, M, H, D).requires_grad_(), _normal(22, M, G, D).requires_grad_()
    gq, gk = (1 + _normal(23, D, scale=0.2)).requires_grad_(), (1 + _normal(24, D, scale=0.2)).requires_grad_()
    pos = torch.arange(M, device='cuda') * 37
    w = _normal(25, M, H, D)
    yq, _ = ops.qk_norm_rope(x, k, gq, gk, pos)
    dx, dk, dgq, dgk = torch.autograd.grad((yq * w).sum(), [x, k, gq, gk])
    assert not dk.any() and not dgk.any()
    # central differences of the fp32 operator along a direction: step h, error h^2 |f'''| + rounding / h
    for leaf, grad in ((x, dx), (gq, dgq)):
        d = _normal(26, *leaf.shape)
        h = 2.0 ** -8

        def f(t):
            args = [x.detach(), k.detach(), gq.detach(), gk.detach()]
            args[0 if leaf is x else 2] = t
            return (ops.qk_norm_rope(*args, pos)[0].double() * w.double()).sum()
        diff = (f(leaf.detach() + h * d) - f(leaf.detach() - h * d)) / (2 * h)
        exact = (grad.double() * d.double()).sum()
        assert abs(diff - exact) <= 2e-3 * (grad.double() * d.double()).abs().sum() + 1e-3


# ---- attention ----------------------------------------------------------------------------------------------------------------------
LENGTHS = [([1], [1]), ([31, 0, 32, 33], [31, 0, 32, 33]), ([63, 64, 65, 1], [63, 64, 65, 1]), ([127, 129, 300], [127, 129, 300]),
           ([5, 64, 1], [133, 64, 260]),                       # the queries are the last frames of longer clips
           ([140, 3, 40, 7], [9, 0, 39, 7])]                   # first rows, or whole clips, that see nothing


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('H,G,D', [(2, 2, 64), (6, 2, 128), (5, 1, 64), (4, 4, 128)])
@pytest.mark.parametrize('ql,kl', LENGTHS)
@pytest.mark.parametrize('causal', [True, False])
def test_attention(ops, eng, dtype, H, G, D, ql, kl, causal):
    q, k, v = _qkv(31, sum(ql), sum(kl), H, G, D, dtype)
    dout = _normal(35, sum(ql), H, D, dtype=dtype)
    batch, kv = _batch(ql), _batch(kl)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.causal_attention(*leaves, batch, kv_batch=kv, causal_mask=causal)
    grads = torch.autograd.grad(out, leaves, dout)
    assert torch.equal(eng.causal_attention(q, k, v, batch, kv_batch=kv, causal_mask=causal), out)
    w = oracle.attention(q, k, v, ql, kl, causal, dout=dout)
    for i, (name, got) in enumerate(zip(('out', 'dq', 'dk', 'dv'), (out.detach(), *grads))):
        oracle.check(got, w[2 * i], w[2 * i + 1], name)
    again = torch.autograd.grad(ops.causal_attention(*leaves, batch, kv_batch=kv, causal_mask=causal), leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('H,G,D,clips', [(16, 16, 64, 40), (48, 16, 128, 40), (4, 2, 64, 640)])
@pytest.mark.parametrize('ql,kl', LENGTHS + [([513, 70, 129], [513, 70, 129])])
@pytest.mark.parametrize('causal', [True, False])
def test_attention_among_empty_clips(ops, eng, dtype, H, G, D, clips, ql, kl, causal):
    """Clips without frames, fewer and more than the block map takes in one wave, and more heads than one workgroup's worth."""
    ql, kl = ql + [0] * clips, kl + [0] * clips
    q, k, v = _qkv(131, sum(ql), sum(kl), H, G, D, dtype)
    dout = _normal(135, sum(ql), H, D, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.causal_attention(*leaves, _batch(ql), kv_batch=_batch(kl), causal_mask=causal)
    grads = torch.autograd.grad(out, leaves, dout)
    w = oracle.attention(q, k, v, ql, kl, causal, dout=dout)
    for i, (name, got) in enumerate(zip(('out', 'dq', 'dk', 'dv'), (out.detach(), *grads))):
        oracle.check(got, w[2 * i], w[2 * i + 1], name)
    again = torch.autograd.grad(ops.causal_attention(*leaves, _batch(ql), kv_batch=_batch(kl), causal_mask=causal), leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize('B', [2, 63, 64, 65, 150])
@pytest.mark.parametrize('past', [False, True])
def test_attention_of_many_clips(ops, B, past):
    """Every tile of every clip is worked on once, whatever the number of clips and their lengths."""
    rng = np.random.default_rng(B)
    ql = [int(n) for n in rng.choice([0, 1, 5, 127, 128, 129, 200, 260], B)]
    kl = [n + int(rng.choice([0, 3, 128, 140])) for n in ql] if past else ql
    H, G, D = 3, 1, 64
    q, k, v = _qkv(37, sum(ql), sum(kl), H, G, D, torch.bfloat16)
    dout = _normal(39, sum(ql), H, D, dtype=torch.bfloat16)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.causal_attention(*leaves, _batch(ql), kv_batch=_batch(kl))
    grads = torch.autograd.grad(out, leaves, dout)
    w = oracle.attention(q, k, v, ql, kl, dout=dout)
    for i, (name, got) in enumerate(zip(('out', 'dq', 'dk', 'dv'), (out.detach(), *grads))):
        oracle.check(got, w[2 * i], w[2 * i + 1], name)


@pytest.mark.parametrize('dtype', TYPES)
def test_attention_of_slices_and_scale(ops, eng, dtype):
    lens, H, G, D = [70, 1, 150], 4, 2, 64
    M = sum(lens)
    fused = _normal(41, M, (H + 2 * G) * D, dtype=dtype)
    leaf = fused.detach().requires_grad_()
    q, k, v = leaf.split([H * D, G * D, G * D], dim=1)
    out = ops.causal_attention(q, k, v, _batch(lens), scale=0.3, head_dim=D)
    assert out.shape == (M, H * D)
    dout = _normal(42, M, H * D, dtype=dtype)
    d, = torch.autograd.grad(out, leaf, dout)
    parts = [t.view(M, -1, D) for t in fused.split([H * D, G * D, G * D], dim=1)]
    w = oracle.attention(*parts, lens, lens, scale=0.3, dout=dout.view(M, H, D))
    oracle.check(out.detach().view(M, H, D), w[0], w[1], 'out')
    got = [t.view(M, -1, D) for t in d.split([H * D, G * D, G * D], dim=1)]
    for i, (name, x) in enumerate(zip(('dq', 'dk', 'dv'), got)):
        oracle.check(x, w[2 + 2 * i], w[3 + 2 * i], name)
    # one key / value head expanded over the rows' heads (stride 0), and heads before rows
    ke, ve = (t[:, :1].expand(M, G, D) for t in parts[1:])
    e = eng.causal_attention(parts[0], ke, ve, _batch(lens))
    assert torch.equal(e, eng.causal_attention(parts[0], ke.contiguous(), ve.contiguous(), _batch(lens)))
    t = parts[0].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(eng.causal_attention(t, parts[1], parts[2], _batch(lens)), eng.causal_attention(parts[0], parts[1], parts[2], _batch(lens)))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('clips', [0, 640])
def test_attention_large_logits(ops, dtype, D, clips):
    """Logits of some hundreds, one key far above the rest, rows whose maximum arrives in the last tile."""
    lens, H, G = [333] + [0] * clips, 2, 1
    q, k, v = _qkv(51, 333, 333, H, G, D, dtype)
    q, k = q * 4, k * 4
    k[200] *= 3
    q, k = q.to(dtype), k.to(dtype)
    out = ops.causal_attention(q, k, v, _batch(lens))
    oracle.check(out, *oracle.attention(q, k, v, lens, lens), 'out')


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize('clips', [0, 640])
def test_attention_is_blind_to_masked_places(eng, dtype, D, bad, clips):
    """Whatever stands at a later frame of the clip, in another clip or behind the last one does not reach an earlier frame."""
    lens, H, G = [97, 40, 66] + [0] * clips, 4, 2
    M = sum(lens)
    q, k, v = _qkv(61, M + 9, M + 9, H, G, D, dtype)
    clean = eng.causal_attention(q[:M], k[:M], v[:M], _batch(lens))
    for at in (5, 50, 96, 97 + 39, 97 + 40, M - 1):
        k2, v2 = k.clone(), v.clone()
        k2[at] = bad
        v2[at] = bad
        k2[M:] = bad
        v2[M:] = bad
        got = eng.causal_attention(q[:M], k2[:M], v2[:M], _batch(lens))
        end = 97 if at < 97 else 97 + 40 if at < 97 + 40 else M
        untouched = torch.ones(M, dtype=torch.bool, device='cuda')
        untouched[at:end] = False
        tol = 2 ** -20 if dtype == torch.float32 else 4 * oracle.half_step(dtype)
        # the block that holds the value is summed in another order there: equal to a rounding of the operand type per probability
        assert torch.isfinite(got[untouched]).all()
        assert (got[untouched].double() - clean[untouched].double()).abs().max() <= tol * v[:M].double().abs().max()
        if math.isnan(bad):
            assert torch.isnan(got[at:end]).all()


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('frames,past', [(2, 0), (3, 0), (1, 1), (2, 3000)])
def test_gradients_of_short_clips_keep_their_precision(ops, dtype, D, frames, past):
    """A row of few keys: dP - D is far smaller than its two terms, so D must not come from the rounded output alone.  Three independent roundings (the
    probabilities, dS, the result), each of a relative mean square of at most (half step)^2 / 3, leave a relative mean square of (half step)^2."""
    ql, H = [frames] * 60, 2
    kl = [frames + past] * 60
    q, k, v = _qkv(141, sum(ql), sum(kl), H, H, D, dtype)
    dout = _normal(145, sum(ql), H, D, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.causal_attention(*leaves, _batch(ql), kv_batch=_batch(kl)), leaves, dout)
    w = oracle.attention(q, k, v, ql, kl, dout=dout)
    for name, got, want in zip(('dq', 'dk', 'dv'), grads, w[2::2]):
        off = ((got.double() - want).pow(2).sum() / want.pow(2).sum()).sqrt().item()
        assert off < oracle.half_step(dtype), (name, off)


@pytest.mark.parametrize('magnitude', [1e-7, 1e-3, 1.0, 3e4])
@pytest.mark.parametrize('clips', [0, 640])
def test_half_precision_gradients_of_any_magnitude(ops, magnitude, clips):
    """f16 holds dO itself to a step; dS, far below or above f16's range, must not lose more."""
    lens, H, G, D = [200, 65] + [0] * clips, 4, 2, 64
    M = sum(lens)
    q, k, v = _qkv(71, M, M, H, G, D, torch.float16)
    dout = (_normal(75, M, H, D) * magnitude).half()
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(ops.causal_attention(*leaves, _batch(lens)), leaves, dout)
    w = oracle.attention(q, k, v, lens, lens, dout=dout)
    for i, name in enumerate(('dq', 'dk', 'dv')):
        want, tol = w[2 + 2 * i], w[3 + 2 * i]
        keep = want.abs() < 65000                                  # what f16 cannot hold is infinite, as anywhere
        oracle.check(grads[i], want.masked_fill(~keep, math.nan), tol, name)


def test_attention_long_rows_past_32_bit_offsets(eng):
    """Rows 16 KiB apart: the clip's last row lies past 2^31 elements."""
    n, H, G, D = 300000, 2, 1, 64
    big = torch.empty(n, 8192, dtype=torch.bfloat16, device='cuda')
    k, v = big[:, :D].unsqueeze(1), big[:, D:2 * D].unsqueeze(1)
    k.copy_(_normal(81, n, 1, D))
    v.copy_(_normal(82, n, 1, D))
    assert k[-1].storage_offset() > 2 ** 31
    q = _normal(83, 100, H, D, dtype=torch.bfloat16)
    out = eng.causal_attention(q, k, v, _batch([100]), kv_batch=_batch([n]))
    oracle.check(out, *oracle.attention(q, k, v, [100], [n]), 'out')
    got = eng.attention_step(q[99:], k[None], v[None], torch.tensor([n], dtype=torch.int32, device='cuda'))
    oracle.check(got, *(x[99:] for x in oracle.attention(q, k, v, [100], [n])), 'step')


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('H,G,D', [(4, 1, 64), (2, 2, 128)])
def test_few_queries_over_many_keys(ops, eng, dtype, H, G, D):
    """The keys are cut into parts here (and the queries of a key tile in the backward): unequal clips, parts that see nothing, values that are not finite."""
    import some_amd._lib as _lib
    ql, kl = [130, 3, 1, 40], [3001, 2, 1500, 40]
    assert _lib.load().some_op_causal_attention_bytes(None, TYPES.index(dtype), H, G, D, 4, sum(ql), sum(kl)) > 0
    q, k, v = _qkv(84, sum(ql), sum(kl), H, G, D, dtype)
    dout = _normal(87, sum(ql), H, D, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.causal_attention(*leaves, _batch(ql), kv_batch=_batch(kl))
    grads = torch.autograd.grad(out, leaves, dout)
    w = oracle.attention(q, k, v, ql, kl, dout=dout)
    for i, (name, got) in enumerate(zip(('out', 'dq', 'dk', 'dv'), (out.detach(), *grads))):
        oracle.check(got, w[2 * i], w[2 * i + 1], name)
    v2 = v.clone()
    v2[2999] = math.nan                                            # seen by the clip's last two queries
    got = eng.causal_attention(q, k, v2, _batch(ql), kv_batch=_batch(kl))
    oracle.check(got[:128], w[0][:128], w[1][:128], 'before')
    assert torch.isnan(got[128:130]).all()
    oracle.check(got[130:], w[0][130:], w[1][130:], 'other clips')


def test_rows_behind_the_last_clip_stay(eng):
    """Through the C ABI: offsets that end before the arrays do."""
    import some_amd._lib as _lib
    lens, H, G, D, extra = [40, 100], 2, 1, 64, 13
    M = sum(lens)
    q, k, v = _qkv(91, M + extra, M + extra, H, G, D, torch.bfloat16)
    out, rest = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
    lse = torch.full((H, M + extra), 7.0, device='cuda')
    b = _batch(lens)
    lib, h = _lib.fast(), eng.handle.value
    st = torch.cuda.current_stream().cuda_stream
    s3 = lambda t: (t.data_ptr(), t.stride(0), t.stride(1))          # noqa: E731
    off = b.frame_offsets_dev.data_ptr()
    _lib.check(h, lib.some_op_causal_attention(h, 2, D, *s3(q), H, *s3(k), *s3(v), G, off, off, b.B, M + extra, M + extra, 1, 0.125, *s3(out), rest.data_ptr(), lse.data_ptr(), None, 0, st))
    assert (out[M:] == 7).all() and (rest[M:] == 7).all() and (lse[:, M:] == 7).all()
    assert torch.equal(out[:M], eng.causal_attention(q[:M], k[:M], v[:M], b))
    dout, work = torch.ones_like(q), torch.empty(1 << 24, dtype=torch.uint8, device='cuda')
    d = [torch.full_like(t, 7.0) for t in (q, k, v)]
    _lib.check(h, lib.some_train_causal_attention_bwd(h, 2, D, *s3(q), H, *s3(k), *s3(v), G, off, off, b.B, M + extra, M + extra, 1, 0.125, *s3(out), rest.data_ptr(), lse.data_ptr(),
                                                      *s3(dout), *s3(d[0]), *s3(d[1]), *s3(d[2]), work.data_ptr(), work.numel(), st))
    assert all((t[M:] == 7).all() for t in d) and not any((t[:M] == 7).all() for t in d)


# ---- the single-frame step --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('H,G,D', [(8, 8, 64), (6, 2, 128), (5, 1, 64), (40, 1, 128)])
@pytest.mark.parametrize('lens,cap', [([1], 1), ([0, 1, 31, 32, 33], 40), ([129, 0, 1000, 517], 1111), ([4097], 5000)])
def test_step(eng, dtype, H, G, D, lens, cap):
    B = len(lens)
    q = _normal(101, B, H, D, dtype=dtype)
    kc, vc = _normal(102, B, cap, G, D, dtype=dtype), _normal(103, B, cap, G, D, dtype=dtype)
    for b, n in enumerate(lens):                                    # what lies behind a stream's length is not read
        kc[b, n:] = math.nan
        vc[b, n:] = math.inf
    k, v = (torch.cat([c[b, :n] for b, n in enumerate(lens)]) for c in (kc, vc))
    want = oracle.attention(q, k, v, [1] * B, lens)
    n = torch.tensor(lens, dtype=torch.int32, device='cuda')
    got = eng.attention_step(q, kc, vc, n)
    oracle.check(got, *want, 'step')
    assert torch.equal(got, eng.attention_step(q, kc, vc, n))
    oracle.check(eng.attention_step(q, kc, vc, n, max_length=max(lens)), *want, 'step with max_length')
    # caches laid out [B, G, T, D], the query a slice
    kt, vt = (c.transpose(1, 2).contiguous().transpose(1, 2) for c in (kc, vc))
    qs = torch.cat([q, q], 1)[:, :H]
    assert torch.equal(got, eng.attention_step(qs, kt, vt, n))


def test_step_cuts_lengths_to_the_cache(eng):
    q, c = _normal(111, 2, 4, 64), _normal(112, 2, 50, 2, 64)
    n = torch.tensor([70, -3], dtype=torch.int32, device='cuda')
    got = eng.attention_step(q, c, c, n)
    assert torch.equal(got[:1], eng.attention_step(q[:1], c[:1], c[:1], torch.tensor([50], dtype=torch.int32, device='cuda')))
    assert not got[1].any()
    assert not eng.attention_step(q, c, c, n, max_length=0).any()
    assert torch.equal(eng.attention_step(q, c, c, n, max_length=20)[:1], eng.attention_step(q, c[:, :20].contiguous(), c[:, :20].contiguous(), n)[:1])


# ---- together ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES)
def test_a_stream_of_frames_equals_the_whole_clip(eng, dtype):
    """norm + rotation + attention of whole clips = the same clips in a first chunk, a second one over the cache, then frame by frame."""
    from some_amd.causal import frame_positions
    lens, first, second, H, G, D = [50, 21], 13, 5, 4, 2, 64
    M, B, cap = sum(lens), 2, 64
    q, k, v = _qkv(121, M, M, H, G, D, dtype)
    gq, gk = 1 + _normal(124, D, scale=0.2), 1 + _normal(125, D, scale=0.2)
    batch = _batch(lens)
    yq, yk = eng.qk_norm_rope(q, k, gq, gk, frame_positions(batch))
    whole = eng.causal_attention(yq, yk, v, batch)
    w, tol = oracle.attention(yq, yk, v, lens, lens)
    oracle.check(whole, w, tol, 'whole')
    start = [0, lens[0]]
    kc, vc = torch.empty(B, cap, G, D, dtype=dtype, device='cuda'), torch.empty(B, cap, G, D, dtype=dtype, device='cuda')
    done = [0, 0]

    def rows(n):
        return torch.cat([torch.arange(start[b] + done[b], start[b] + done[b] + n[b]) for b in range(B)]).cuda()

    for n in ([first, first], [second, 2]):
        r = rows(n)
        pos = torch.cat([torch.arange(done[b], done[b] + n[b]) for b in range(B)]).cuda()
        cq, ck = eng.qk_norm_rope(q[r], k[r], gq, gk, pos)
        assert torch.equal(cq, yq[r]) and torch.equal(ck, yk[r])
        at = 0
        for b in range(B):
            kc[b, done[b]:done[b] + n[b]], vc[b, done[b]:done[b] + n[b]] = ck[at:at + n[b]], v[r][at:at + n[b]]
            done[b] += n[b]
            at += n[b]
        kk, vv = (torch.cat([c[b, :done[b]] for b in range(B)]) for c in (kc, vc))
        out = eng.causal_attention(cq, kk, vv, _batch(n), kv_batch=_batch(done))
        oracle.check(out, w[r], tol[r], 'chunk')
    while done[1] < lens[1]:
        r = rows([1, 1])
        pos = torch.tensor(done, device='cuda')
        cq, ck = eng.qk_norm_rope(q[r], k[r], gq, gk, pos)
        for b in range(B):
            kc[b, done[b]], vc[b, done[b]] = ck[b], v[r[b]]
            done[b] += 1
        out = eng.attention_step(cq, kc, vc, torch.tensor(done, dtype=torch.int32, device='cuda'))
        oracle.check(out, w[r], tol[r], 'frame')


def _layer(ops, x, wq, wk, wv, wo, gq, gk, batch, pos):
    q, k, v = ops.linear(x, wq), ops.linear(x, wk), ops.linear(x, wv)
    q, k = ops.qk_norm_rope(q, k, gq, gk, pos)
    return ops.linear(ops.causal_attention(q, k, v, batch, head_dim=64), wo)


def test_training_layer_on_autograd_and_tape(ops):
    """A causal attention layer from the framework's operators: the trainer's tape gives autograd's gradients bit for bit, and gradient sinks receive them."""
    from some_amd.causal import frame_positions
    from some_amd.training.ops import Tape
    lens, C, H, G = [70, 129], 128, 4, 2
    M = sum(lens)
    batch = _batch(lens)
    pos = frame_positions(batch)
    x = _normal(131, M, C)
    shapes = [(H * 64, C), (G * 64, C), (G * 64, C), (C, H * 64)]
    def params():                                                                           # noqa: E306
        ps = [_normal(132 + i, *s, scale=C ** -0.5).requires_grad_() for i, s in enumerate(shapes)]
        return ps + [(1 + _normal(140 + i, 64, scale=0.1)).requires_grad_() for i in range(2)]
    dy = _normal(150, M, C)
    a = params()
    ya = _layer(ops, x, *a, batch, pos)
    ya.backward(dy)
    b = params()
    for p in b:
        p.grad = torch.zeros_like(p)
    told = []
    tape = ops.tape = Tape(ops)
    try:
        ops.register_grad_sinks(b[4:], lambda p: told.append(id(p)))
        with torch.no_grad():
            yb = _layer(ops, x, *b, batch, pos)
        tape.backward([(yb, dy)])
    finally:
        ops.tape = None
        ops.register_grad_sinks([])
    assert torch.equal(ya, yb)
    for p, r in zip(a, b):
        assert torch.equal(p.grad, r.grad)
    assert id(b[4]) in told and id(b[5]) in told
    # the definition, differentiated in 64 bits
    d = [p.detach().double().requires_grad_() for p in a]
    xd = x.double()

    def rope(t, g):
        t = t.view(M, -1, 64)
        t = t / (t.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * g
        ang = pos.double()[:, None, None] * 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64, device='cuda') / 64)
        u, w = t[..., :32], t[..., 32:]
        return torch.cat([u * ang.cos() - w * ang.sin(), w * ang.cos() + u * ang.sin()], -1)
    q, k, v = rope(xd @ d[0].t(), d[4]), rope(xd @ d[1].t(), d[5]), (xd @ d[2].t()).view(M, G, 64)
    outs, at = [], 0
    for n in lens:
        s = torch.einsum('ihd,jhd->hij', q[at:at + n], k[at:at + n].repeat_interleave(H // G, 1)) / 8
        s = s.masked_fill(torch.ones(n, n, device='cuda', dtype=torch.bool).triu(1), -math.inf)
        outs.append(torch.einsum('hij,jhd->ihd', s.softmax(-1), v[at:at + n].repeat_interleave(H // G, 1)))
        at += n
    yd = torch.cat(outs).reshape(M, -1) @ d[3].t()
    yd.backward(dy.double())
    for got, want in [(ya, yd)] + [(p.grad, r.grad) for p, r in zip(a, d)]:
        # the framework's own fp32-equivalent linears (2^-21 per product) bound the chain: 2e-5 of the scale, as in the tests of the operators
        assert (got.double() - want).abs().max() <= 2e-5 * want.abs().max()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_captured_and_replayed(ops, eng, dtype):
    """Serving calls and a training step captured into graphs: replays with new inputs, eager work between them, equal the eager calls."""
    lens, H, G, D = [65, 200], 4, 2, 64
    M = sum(lens)
    batch = _batch(lens)
    pos = torch.arange(M, device='cuda')
    gq, gk = 1 + _normal(161, D, scale=0.2), 1 + _normal(162, D, scale=0.2)
    ln = torch.tensor([900, 333], dtype=torch.int32, device='cuda')
    buf = list(_qkv(163, M, M, H, G, D, dtype)) + [_normal(166, 2, H, D, dtype=dtype), _normal(167, 2, 1000, G, D, dtype=dtype), _normal(168, 2, 1000, G, D, dtype=dtype)]
    dout = _normal(169, M, H, D, dtype=dtype)

    def step(q, k, v, sq, kc, vc):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        g1, g2 = gq.detach().requires_grad_(), gk.detach().requires_grad_()
        yq, yk = ops.qk_norm_rope(q, k, g1, g2, pos)
        out = ops.causal_attention(yq, yk, v, batch)
        grads = torch.autograd.grad(out, [q, k, v, g1, g2], dout)
        with torch.no_grad():
            return [out.detach(), *grads, *eng.qk_norm_rope(q, k, gq, gk, pos), eng.attention_step(sq, kc, vc, ln)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*buf)
    side.synchronize()
    graphs = []
    for _ in range(2):                                             # two graphs of the same calls: each its own workspaces
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            graphs.append((g, step(*buf)))
    for i in range(3):
        for j, b in enumerate(buf):
            b.copy_(_normal(200 + 10 * i + j, *b.shape, dtype=dtype))
        eager = step(*buf)
        torch.cuda.synchronize()
        for g, outs in graphs:
            g.replay()
        for g, outs in graphs:
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(eager, outs))


def test_another_stream(ops, eng):
    lens, H, G, D = [333], 8, 2, 64
    q, k, v = _qkv(181, 333, 333, H, G, D, torch.bfloat16)
    want = eng.causal_attention(q, k, v, _batch(lens))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b = _batch(lens)
    with torch.cuda.stream(s):
        got = eng.causal_attention(q, k, v, b)
        step = eng.attention_step(q[-1:], k[None], v[None], torch.tensor([333], dtype=torch.int32, device='cuda'))
    s.synchronize()
    assert torch.equal(got, want)
    oracle.check(step, *(t[-1:] for t in oracle.attention(q, k, v, lens, lens)), 'step')


def test_empty_batches(eng, ops):
    q, k, v = _qkv(191, 0, 0, 4, 2, 64, torch.float32)
    for lens in ([], [0, 0]):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.causal_attention(*leaves, _batch(lens))
        out.sum().backward()
        assert out.shape == q.shape and leaves[1].grad.shape == k.shape
    k, v = _normal(192, 30, 2, 64), _normal(193, 30, 2, 64)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.causal_attention(*leaves, _batch([0]), kv_batch=_batch([30]))         # keys nobody asks for: zero gradients
    out.sum().backward()
    assert not leaves[1].grad.any() and not leaves[2].grad.any()
    n = torch.zeros(0, dtype=torch.int32, device='cuda')
    assert eng.attention_step(q[:0], k[None][:0], v[None][:0], n).shape == (0, 4, 64)


def test_refusals_on_the_device(eng, ops):
    q, k, v = _qkv(195, 10, 10, 4, 2, 64, torch.float32)
    b = _batch([10])
    with pytest.raises(RuntimeError, match='not differentiable'):
        eng.causal_attention(q.requires_grad_(), k, v, b)
    q = q.detach()
    with pytest.raises(ValueError, match='on cpu'):
        eng.causal_attention(q, k, v.cpu(), b)
    with pytest.raises(ValueError, match='copy per frame'):
        c = torch.zeros(1, 5, 2, 65, device='cuda')[..., 1:]
        eng.attention_step(q[:1], c, c, torch.tensor([3], dtype=torch.int32, device='cuda'))
    with pytest.raises(RuntimeError, match='twice|does not require grad'):
        x = q.requires_grad_()
        g, = torch.autograd.grad(ops.causal_attention(x, k, v, b).sum(), x, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('clips', [0, 640])
def test_gradients_are_blind_to_masked_places(ops, dtype, D, clips):
    """A value that is not finite makes the gradients of what it meets non-finite - and of nothing else."""
    lens, H, G = [97, 66] + [0] * clips, 4, 2
    M = sum(lens)
    q, k, v = _qkv(301, M, M, H, G, D, dtype)
    dout = _normal(305, M, H, D, dtype=dtype)
    batch = _batch(lens)

    def grads(q, k, v, dout):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(ops.causal_attention(*leaves, batch), leaves, dout)
    clean = grads(q, k, v, dout)
    scale = [c.double().abs().max() * 8 * max(oracle.half_step(dtype), 2.0 ** -22) for c in clean]
    for at, end in ((40, 97), (97 + 33, M)):
        begin = end - (97 if end == 97 else 66)
        # dO of frame `at`: frames after it keep their key gradients, every other frame its query gradient
        d2 = dout.clone()
        d2[at] = math.inf
        got = grads(q, k, v, d2)
        rows = torch.ones(M, dtype=torch.bool, device='cuda')
        rows[at] = False
        keys = torch.ones(M, dtype=torch.bool, device='cuda')
        keys[begin:at + 1] = False
        for x, c, m, s in zip(got, clean, (rows, keys, keys), scale):
            assert torch.isfinite(x[m]).all() and (x[m].double() - c[m].double()).abs().max() <= s
        # key and value of frame `at`: the frames before it keep their query gradients
        k2, v2 = k.clone(), v.clone()
        k2[at] = math.nan
        v2[at] = math.nan
        dq = grads(q, k2, v2, dout)[0]
        before = torch.ones(M, dtype=torch.bool, device='cuda')
        before[at:end] = False
        assert torch.isfinite(dq[before]).all() and (dq[before].double() - clean[0][before].double()).abs().max() <= scale[0]


@pytest.mark.parametrize('dtype', TYPES)
def test_rows_behind_the_last_clip_stay_where_parts_are_joined(eng, dtype):
    """Few queries over many keys, offsets that begin and end inside the arrays: the joins write the clips' rows alone."""
    import some_amd._lib as _lib
    code, H, G, D, n, t, edge = TYPES.index(dtype), 4, 2, 64, 40, 3000, 5
    lib, h = _lib.fast(), eng.handle.value
    q, k, v = _qkv(401, n + 2 * edge, t + 2 * edge, H, G, D, dtype)
    dout = _normal(405, n + 2 * edge, H, D, dtype=dtype)
    qo = torch.tensor([edge, edge + 1, edge + n], dtype=torch.int32, device='cuda')
    ko = torch.tensor([edge, edge + 1000, edge + t], dtype=torch.int32, device='cuda')
    M, N = len(q), len(k)
    s3 = lambda x: (x.data_ptr(), x.stride(0), x.stride(1))                                   # noqa: E731
    out, rest, lse = torch.full_like(q, 7.0), torch.full_like(q, 7.0), torch.full((H, M), 7.0, device='cuda')
    nb = lib.some_op_causal_attention_bytes(h, code, H, G, D, 2, M, N)
    assert nb > 0
    work = torch.full((lib.some_train_causal_attention_bytes(h, code, H, G, D, 2, M, N),), 255, dtype=torch.uint8, device='cuda')
    st = torch.cuda.current_stream().cuda_stream
    _lib.check(h, lib.some_op_causal_attention(h, code, D, *s3(q), H, *s3(k), *s3(v), G, qo.data_ptr(), ko.data_ptr(), 2, M, N, 1, 0.125, *s3(out), rest.data_ptr(),
                                               lse.data_ptr(), work.data_ptr(), work.numel(), st))
    d = [torch.full_like(x, 7.0) for x in (q, k, v)]
    work.fill_(255)
    _lib.check(h, lib.some_train_causal_attention_bwd(h, code, D, *s3(q), H, *s3(k), *s3(v), G, qo.data_ptr(), ko.data_ptr(), 2, M, N, 1, 0.125, *s3(out), rest.data_ptr(),
                                                      lse.data_ptr(), *s3(dout), *s3(d[0]), *s3(d[1]), *s3(d[2]), work.data_ptr(), work.numel(), st))
    for x in (out, *d) if dtype == torch.float32 else (out, rest, *d):
        assert (x[:edge] == 7).all() and (x[-edge:] == 7).all()
    assert (lse[:, :edge] == 7).all() and (lse[:, -edge:] == 7).all()
    inner = [x[edge:-edge] for x in (q, k, v, dout)]
    w = oracle.attention(*inner[:3], [1, n - 1], [1000, t - 1000], dout=inner[3])
    for i, (name, got) in enumerate(zip(('out', 'dq', 'dk', 'dv'), (out, *d))):
        oracle.check(got[edge:-edge], w[2 * i], w[2 * i + 1], name)


def test_norm_rope_past_32_bit_offsets(ops):
    n, H, D = 700, 2, 64
    big = torch.empty(n * 4_000_000, dtype=torch.bfloat16, device='cuda')
    q = big.as_strided((n, H, D), (4_000_000, D, 1))
    k = big.as_strided((n, 1, D), (4_000_000, D, 1), H * D)
    q.copy_(_normal(411, n, H, D))
    k.copy_(_normal(412, n, 1, D))
    assert q[-1].storage_offset() > 2 ** 31
    g = 1 + _normal(413, D, scale=0.2)
    pos = torch.arange(n, device='cuda')
    dy = _normal(414, n, H, D, dtype=torch.bfloat16)
    leaves = [q.detach().requires_grad_(), g.requires_grad_()]
    yq, yk = ops.qk_norm_rope(leaves[0], k, g, g, pos)
    dq, dg = torch.autograd.grad(yq, leaves, dy)
    w = oracle.norm_rope(q, g, pos, dy=dy)
    oracle.check(yq.detach(), w[0], w[1], 'q')
    oracle.check(yk.detach(), *oracle.norm_rope(k, g, pos), 'k')
    oracle.check(dq, w[2], w[3], 'dq')
    oracle.check(dg, w[4], w[5], 'dgamma')                         # the keys' share of the common gain is zero: no cotangent


def test_one_gain_for_both_and_one_array_for_keys_and_values(ops):
    """The same leaf twice in a call: its gradients add up."""
    M, H, G, D = 130, 4, 2, 64
    q, k, _ = _qkv(421, M, M, H, G, D, torch.float32)
    g, pos = 1 + _normal(424, D, scale=0.2), torch.arange(M, device='cuda')
    dq, dk = _normal(425, M, H, D), _normal(426, M, G, D)
    a = g.clone().requires_grad_()
    got, = torch.autograd.grad(ops.qk_norm_rope(q, k, a, a, pos), a, (dq, dk))
    b, c = g.clone().requires_grad_(), g.clone().requires_grad_()
    want = torch.autograd.grad(ops.qk_norm_rope(q, k, b, c, pos), (b, c), (dq, dk))
    assert torch.equal(got, want[0] + want[1])
    a = k.clone().requires_grad_()
    got, = torch.autograd.grad(ops.causal_attention(q, a, a, _batch([M])), a, dq)
    b, c = k.clone().requires_grad_(), k.clone().requires_grad_()
    want = torch.autograd.grad(ops.causal_attention(q, b, c, _batch([M])), (b, c), dq)
    assert torch.equal(got, want[0] + want[1])


@pytest.mark.parametrize('cap', [300, 5000])
def test_step_replayed_with_other_lengths(eng, cap):
    """Lengths are read on the device: one capture serves a stream from its first frame to a full cache."""
    B, H, G, D = 3, 8, 2, 128
    q, kc, vc = _normal(431, B, H, D, dtype=torch.float16), _normal(432, B, cap, G, D, dtype=torch.float16), _normal(433, B, cap, G, D, dtype=torch.float16)
    ln = torch.tensor([1, 1, 1], dtype=torch.int32, device='cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eng.attention_step(q, kc, vc, ln)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = eng.attention_step(q, kc, vc, ln)
    for lens in ([1, 0, 2], [cap, cap - 1, 129], [0, 0, 0], [33, cap, 257]):
        ln.copy_(torch.tensor(lens, dtype=torch.int32))
        eager = eng.attention_step(q, kc, vc, ln)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        kk, vv = (torch.cat([c[b, :lens[b]] for b in range(B)]) for c in (kc, vc))
        oracle.check(eager, *oracle.attention(q, kk, vv, [1] * B, lens), str(lens))


def test_two_streams_at_once(ops, eng):
    """Calls that overlap on two streams share nothing: each gives what it gives alone."""
    cases = []
    for i, (lens, H, G) in enumerate((([1500, 900], 4, 1), ([2000], 8, 2))):
        q, k, v = _qkv(441 + 10 * i, sum(lens), sum(lens), H, G, 64, torch.bfloat16)
        dout = _normal(445 + 10 * i, sum(lens), H, 64, dtype=torch.bfloat16)
        cases.append(([t.requires_grad_() for t in (q, k, v)], _batch(lens), dout))

    def run(case):
        leaves, batch, dout = case
        out = ops.causal_attention(*leaves, batch)
        return (out.detach(), *torch.autograd.grad(out, leaves, dout))
    want = [run(c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(run(c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('H,G', [(1024, 1), (1024, 1024), (300, 3), (35, 7)])
def test_many_heads_and_odd_groups(ops, eng, dtype, H, G):
    """Up to 1024 heads: groups larger than a workgroup's 128 queries (a frame then spans tiles), groups that do not divide them, kv heads that do not divide the XCDs."""
    D, ql, kl = 64, [3, 0, 9], [5, 2, 9]
    q, k, v = _qkv(451, sum(ql), sum(kl), H, G, D, dtype)
    dout = _normal(455, sum(ql), H, D, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = ops.causal_attention(*leaves, _batch(ql), kv_batch=_batch(kl))
    grads = torch.autograd.grad(out, leaves, dout)
    w = oracle.attention(q, k, v, ql, kl, dout=dout)
    for i, (name, got) in enumerate(zip(('out', 'dq', 'dk', 'dv'), (out.detach(), *grads))):
        oracle.check(got, w[2 * i], w[2 * i + 1], name)
    cache = [torch.zeros(2, 9, G, D, dtype=dtype, device='cuda') for _ in range(2)]
    for c, t in zip(cache, (k, v)):
        c[0, :5], c[1] = t[:5], t[7:]
    step = eng.attention_step(q[[2, 11]], *cache, torch.tensor([5, 9], dtype=torch.int32, device='cuda'))
    oracle.check(step, w[0][[2, 11]], w[1][[2, 11]], 'step')
    gq, gk, pos = 1 + _normal(456, D, scale=0.2), 1 + _normal(457, D, scale=0.2), torch.arange(sum(ql), device='cuda')
    yq, yk = eng.qk_norm_rope(q, k[:sum(ql)], gq, gk, pos)
    oracle.check(yq, *oracle.norm_rope(q, gq, pos), 'q')
    oracle.check(yk, *oracle.norm_rope(k[:sum(ql)], gk, pos), 'k')


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,H,G', [(7, 4, 2), (3000, 40, 8)])
def test_norm_rope_in_place(ops, eng, dtype, M, H, G):
    """The C entries' outputs may be their inputs."""
    import some_amd._lib as _lib
    D, code, lib, h = 128, TYPES.index(dtype), _lib.fast(), eng.handle.value
    q, k = _normal(461, M, H, D, dtype=dtype), _normal(462, M, G, D, dtype=dtype)
    gq, gk, pos = 1 + _normal(463, D, scale=0.2), 1 + _normal(464, D, scale=0.2), torch.arange(M, device='cuda')
    dq, dk = _normal(465, M, H, D, dtype=dtype), _normal(466, M, G, D, dtype=dtype)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, gq, gk)]
    y = ops.qk_norm_rope(*leaves, pos)
    want = torch.autograd.grad(y, leaves, (dq, dk))
    s3 = lambda t: (t.data_ptr(), t.stride(0), t.stride(1))                                   # noqa: E731
    head = (h, code, D, *s3(q), H, *s3(k), G, M, gq.data_ptr(), gk.data_ptr(), pos.data_ptr(), 1, 10000.0, 1e-6)
    st = torch.cuda.current_stream().cuda_stream
    work = torch.empty(lib.some_train_qk_norm_rope_bytes(h, M, H, G, D), dtype=torch.uint8, device='cuda')
    dgq, dgk = torch.empty_like(gq), torch.empty_like(gk)
    _lib.check(h, lib.some_train_qk_norm_rope_bwd(*head, *s3(dq), *s3(dk), *s3(dq), *s3(dk), dgq.data_ptr(), dgk.data_ptr(), 0, work.data_ptr(), work.numel(), st))
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dgq, dgk), want))
    _lib.check(h, lib.some_op_qk_norm_rope(*head, *s3(q), *s3(k), st))
    assert torch.equal(q, y[0]) and torch.equal(k, y[1])
