"""Causal attention operators at the edges of their arithmetic on a real MI355X, against the 64-bit definitions (tests/causal_oracle.py)."""
import math

import pytest
import torch

import causal_oracle as oracle
from some_amd import _lib
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


def _check_all(got, want):
    for i, (name, x) in enumerate(zip(('out', 'dq', 'dk', 'dv'), got)):
        oracle.check(x.detach(), want[2 * i], want[2 * i + 1], name)


ALONE = [1] * 600                 # so many clips beside the one looked at that nothing is cut into parts


def _whole(dtype, H, G, D, ql, kl):
    assert _lib.load().some_op_causal_attention_bytes(None, TYPES.index(dtype), H, G, D, len(ql), sum(ql), sum(kl)) == 0


# ---- one dominating key -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('n', [16384, 65536])
@pytest.mark.parametrize('gap,spread', [(17.4, 0.05), (18.0, 1.0), (22.0, 0.05)])
@pytest.mark.parametrize('where', ['first', 'last'])
def test_half_precision_rows_with_one_dominating_key(eng, D, n, gap, spread, where):
    """f16: the weights of all other keys together matter where the dominating key's value is small, and each of them is far below f16's normal range
    beside a largest weight of 1."""
    ql, kl = [33] + ALONE, [n] + ALONE
    _whole(torch.float16, 1, 1, D, ql, kl)
    q, k = _normal(1, sum(ql), 1, D, scale=0.01), _normal(2, sum(kl), 1, D, scale=0.01)
    v = 1 + _normal(3, sum(kl), 1, D)
    top = 0 if where == 'first' else n - 100
    q[:, :, 0] = 4.0
    k[:, :, 0] = _normal(4, sum(kl), 1, scale=spread / 4)
    k[top, :, 0] = gap / 4
    v[top] *= 0.01
    q, k, v = q.half(), k.half(), v.half()
    out = eng.causal_attention(q, k, v, _batch(ql), kv_batch=_batch(kl), scale=1.0)
    oracle.check(out, *oracle.attention(q, k, v, ql, kl, scale=1.0), 'out')


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('gaps', [(17.4, 30.0, 60.0), (60.0, 30.0, 17.4), (90.0, 12.0, 90.0), (9.0, 9.0, 9.0)])
def test_half_precision_rows_with_several_dominating_keys(eng, D, gaps):
    """f16: what the weights are taken relative to goes down behind one key and up again at the next."""
    n = 4100
    ql, kl = [33] + ALONE, [n] + ALONE
    _whole(torch.float16, 1, 1, D, ql, kl)
    q, k = _normal(6, sum(ql), 1, D, scale=0.01), _normal(7, sum(kl), 1, D, scale=0.05)
    v = 1 + _normal(8, sum(kl), 1, D)
    q[:, :, 0] = 5.0
    for at, gap in zip((70, 2000, n - 1000), gaps):
        k[at, :, 0] = gap / 5
        v[at] = 0.0
    q, k, v = q.half(), k.half(), v.half()
    out = eng.causal_attention(q, k, v, _batch(ql), kv_batch=_batch(kl), scale=1.0)
    oracle.check(out, *oracle.attention(q, k, v, ql, kl, scale=1.0), 'out')


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('size', [100.0, 2500.0, 13600.0])
@pytest.mark.parametrize('rising', [False, True])
def test_half_precision_rows_of_huge_scores(eng, D, size, rising):
    """f16: scores of 10^3 to 10^7 nats that leave one key a row; the weights keep inside f16's range."""
    n, H = 200, 2
    step = torch.arange(1, n + 1, device='cuda', dtype=torch.float32) * (size / n)
    q, k, v = torch.zeros(n, H, D, device='cuda'), torch.zeros(n, 1, D, device='cuda'), _normal(5, n, 1, D, dtype=torch.float16)
    q[:, :, 7] = size
    k[:, 0, 7] = step if rising else step.flip(0)
    q, k = q.half(), k.half()
    out = eng.causal_attention(q, k, v, _batch([n]), scale=0.125)
    # (the definition's own bound grows with the scores and allows everything here: the weight's rounding and the output's, as the keys lie 6 nats apart at least)
    want = oracle.attention(q, k, v, [n], [n], scale=0.125)[0]
    oracle.check(out, want, 2 * oracle.half_step(torch.float16) * want.abs() + 2.0 ** -11 * v.abs().max().double(), 'out')


@pytest.mark.parametrize('H,G,D', [(2, 2, 64), (5, 1, 128)])
@pytest.mark.parametrize('gap', [12.0, 17.4, 22.0])
@pytest.mark.parametrize('capacity', [520, 3000])
def test_half_precision_step_with_one_dominating_key(eng, H, G, D, gap, capacity):
    """f16: the step's weights as well, whichever tile, wave and chunk the dominating key falls to."""
    tops = [0, 1, 40, 200, 511]
    B, n = len(tops), capacity - 3
    q, kc, vc = _normal(91, B, H, D, scale=0.01), _normal(92, B, capacity, G, D, scale=0.02), 1 + _normal(93, B, capacity, G, D)
    q[..., 0] = 4.0
    for b, at in enumerate(tops):
        kc[b, at, :, 0] = gap / 4
        vc[b, at] = 0.0
    q, kc, vc = q.half(), kc.half(), vc.half()
    got = eng.attention_step(q, kc, vc, torch.full((B,), n, dtype=torch.int32, device='cuda'), scale=1.0)
    k, v = (c[:, :n].reshape(B * n, G, D) for c in (kc, vc))
    oracle.check(got, *oracle.attention(q, k, v, [1] * B, [n] * B, scale=1.0), 'step')


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('gap', [12.0, 22.0, 26.0, 40.0])
@pytest.mark.parametrize('magnitude', [1.0, 1000.0, 20000.0])
def test_half_precision_gradients_of_faint_keys(ops, D, gap, magnitude):
    """f16: the gradient of a value whose weights are all small, over many queries and for gradients of any magnitude."""
    lens = [2000, 129]
    M = sum(lens)
    q, k, v = _normal(11, M, 1, D, scale=0.02), _normal(12, M, 1, D, scale=0.02), _normal(13, M, 1, D)
    q[:, :, 0] = 4.0
    k[0, :, 0] = k[2000, :, 0] = gap / 4
    dout = ((1 + 0.5 * _normal(14, M, 1, D)) * magnitude).half()
    leaves = [t.half().requires_grad_() for t in (q, k, v)]
    out = ops.causal_attention(*leaves, _batch(lens), scale=1.0)
    grads = torch.autograd.grad(out, leaves, dout)
    w = list(oracle.attention(*(t.detach() for t in leaves), lens, lens, scale=1.0, dout=dout))
    for i in (2, 4, 6):
        w[i] = w[i].masked_fill(w[i].abs() >= 65000, math.nan)      # what f16 cannot hold is infinite, as anywhere
    _check_all((out, *grads), w)


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('gap', [17.4, 24.0])
def test_half_precision_gradients_of_a_key_only_one_row_looks_at(ops, D, gap):
    """f16: a key's weight is 1 in its own row, which the loss leaves out, and faint in all others."""
    lens = [3000]
    M = sum(lens)
    q, k, v = _normal(15, M, 2, D, scale=0.02), _normal(16, M, 1, D, scale=0.02), _normal(17, M, 1, D)
    q[:, :, 0] = 4.0
    k[0, :, 0] = -gap / 4
    dout = (1 + 0.5 * _normal(18, M, 2, D)) * 1000
    dout[0] = 0.0
    dout = dout.half()
    leaves = [t.half().requires_grad_() for t in (q, k, v)]
    out = ops.causal_attention(*leaves, _batch(lens), scale=1.0)
    grads = torch.autograd.grad(out, leaves, dout)
    w = list(oracle.attention(*(t.detach() for t in leaves), lens, lens, scale=1.0, dout=dout))
    for i in (2, 4, 6):
        w[i] = w[i].masked_fill(w[i].abs() >= 65000, math.nan)
    # the weights of the 32 rows that share a block (and a power of two) with the key's own row, of both heads: that power brings the weight 1 to 2^11 at least, and
    # f16's smallest step is 2^-24, so each is off by 2^-25 / 2^11 at most
    w[7] = w[7] + 2 * 32 * 2.0 ** -36 * dout.abs().max().double()
    _check_all((out, *grads), w)


# ---- infinities that are seen -------------------------------------------------------------------------------------------------------------
def _infinite_values(v, rows):
    """Copies of v with +inf in channel 3 and -inf in channel 5 of the given rows, and with zeros there."""
    a, b = v.clone(), v.clone()
    for x, p, m in ((a, math.inf, -math.inf), (b, 0.0, 0.0)):
        for r in rows:
            x[r][..., 3] = p
            x[r][..., 5] = m
    return a, b


def _check_infinite(got, want, tol):
    assert (got[..., 3] == math.inf).all() and (got[..., 5] == -math.inf).all()
    rest = [c for c in range(got.shape[-1]) if c not in (3, 5)]
    oracle.check(got[..., rest], want[..., rest], tol[..., rest], 'the other channels')


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('keys', [31, 32, 33, 63, 64, 65, 128, 200])
@pytest.mark.parametrize('queries', [1, 40])
@pytest.mark.parametrize('train', [False, True])
def test_an_infinite_value_every_query_sees(eng, ops, dtype, D, keys, queries, train):
    H, G = 4, 2
    q, k, v = _normal(21, queries, H, D, dtype=dtype), _normal(22, keys, G, D, dtype=dtype), _normal(23, keys, G, D, dtype=dtype)
    inf, fin = _infinite_values(v, [10])
    call = ops if train else eng
    if train:
        q = q.requires_grad_()
    for causal in (False, True) if queries == 1 else (False,):
        got = call.causal_attention(q, k, inf, _batch([queries]), kv_batch=_batch([keys]), causal_mask=causal).detach()
        _check_infinite(got, *oracle.attention(q, k, fin, [queries], [keys], causal))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('H,G,D', [(4, 2, 64), (2, 2, 128), (40, 1, 64)])
@pytest.mark.parametrize('capacity', [40, 1000, 3000])
def test_step_over_a_newest_frame_with_an_infinite_value(eng, dtype, H, G, D, capacity):
    lens = [n for n in (1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 2049, 3000) if n <= capacity]
    B = len(lens)
    q, kc, vc = _normal(31, B, H, D, dtype=dtype), _normal(32, B, capacity, G, D, dtype=dtype), _normal(33, B, capacity, G, D, dtype=dtype)
    inf, fin = _infinite_values(vc, [(b, n - 1) for b, n in enumerate(lens)])
    for b, n in enumerate(lens):
        inf[b, n:] = kc[b, n:] = math.nan
    got = eng.attention_step(q, kc, inf, torch.tensor(lens, dtype=torch.int32, device='cuda'))
    k, v = (torch.cat([c[b, :n] for b, n in enumerate(lens)]) for c in (kc, fin))
    _check_infinite(got, *oracle.attention(q, k, v, [1] * B, lens))


# ---- parts without keys -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', [64, 128])
def test_a_part_without_keys_is_left_zero(eng, dtype, D):
    """Keys in parts, a clip of fewer tiles than parts: what the parts without a tile hand to the join is zeros, not what lay in LDS."""
    ql, kl, H = [64, 64], [8000, 30], 1
    M, N, code = sum(ql), sum(kl), TYPES.index(dtype)
    lib, h = _lib.fast(), eng.handle.value
    q, k, v = (_normal(41 + i, n, H, D, dtype=dtype) for i, n in enumerate((M, N, N)))
    nb = lib.some_op_causal_attention_bytes(h, code, H, H, D, 2, M, N)
    parts = nb // (M * H * (D + 2) * 4)
    assert parts > 2 and parts * M * H * (D + 2) * 4 == nb
    bq, bk = _batch(ql), _batch(kl)                                # (held: the call gets bare addresses of their offsets)
    work, out = torch.full((nb // 4,), 7.0, device='cuda'), torch.empty_like(q)
    s3 = lambda t: (t.data_ptr(), t.stride(0), t.stride(1))                                   # noqa: E731
    _lib.check(h, lib.some_op_causal_attention(h, code, D, *s3(q), H, *s3(k), *s3(v), H, bq.frame_offsets_dev.data_ptr(), bk.frame_offsets_dev.data_ptr(),
                                               2, M, N, 0, 0.125, *s3(out), None, None, work.data_ptr(), nb, torch.cuda.current_stream().cuda_stream))
    sums = work[:parts * M * H * D].view(parts, M, H, D)
    assert not sums[:parts - 1, ql[0]:].any()                      # the one tile of the second clip belongs to the last part
    oracle.check(out, *oracle.attention(q, k, v, ql, kl, False, scale=0.125), 'out')


# ---- long runs of equal frames --------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('n', [16384, 65536])
@pytest.mark.parametrize('values', ['equal', 'unequal'])
def test_long_rows_of_equal_keys(eng, dtype, D, n, values):
    """Silence: all keys alike but one.  Equal weights round the same way, so an error of their sum would grow with their number."""
    ql, kl = [70] + ALONE, [n] + ALONE
    _whole(dtype, 1, 1, D, ql, kl)
    for gain in (0.5, 0.71, 0.9):
        q, k = _normal(51, 1, 1, D).expand(sum(ql), 1, D), _normal(52, 1, 1, D).repeat(sum(kl), 1, 1)
        k[3] += 0.25 * q[0] * gain
        v = _normal(53, 1, 1, D).repeat(sum(kl), 1, 1) if values == 'equal' else 1 + 0.3 * _normal(53, sum(kl), 1, D)
        q, k, v = (t.to(dtype).contiguous() for t in (q, k, v))
        out = eng.causal_attention(q, k, v, _batch(ql), kv_batch=_batch(kl))
        oracle.check(out, *oracle.attention(q, k, v, ql, kl), f'out {gain}')


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('causal', [True, False])
def test_gradients_of_long_runs_of_equal_frames(ops, dtype, D, causal):
    n = 12000
    lens = [n] + ALONE
    M = sum(lens)
    _whole(dtype, 1, 1, D, lens, lens)
    q, k, v, dout = (_normal(61 + i, 1, 1, D).repeat(M, 1, 1).to(dtype) for i in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.causal_attention(*leaves, _batch(lens), causal_mask=causal)
    grads = torch.autograd.grad(out, leaves, dout)
    _check_all((out, *grads), oracle.attention(*(t.detach() for t in leaves), lens, lens, causal, dout=dout))


# ---- scales far from 1 --------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('scale', [2.0 ** -64, 2.0 ** -126, 2.0 ** -130])
def test_a_scale_next_to_nought(ops, dtype, scale):
    """All weights alike: the mean of what a row sees, and gradients to match."""
    lens, H, G, D = [70, 3], 2, 1, 64
    M = sum(lens)
    q, k, v = _normal(71, M, H, D, dtype=dtype), _normal(72, M, G, D, dtype=dtype), _normal(73, M, G, D, dtype=dtype)
    dout = _normal(74, M, H, D, dtype=dtype)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = ops.causal_attention(*leaves, _batch(lens), scale=scale)
    grads = torch.autograd.grad(out, leaves, dout)
    _check_all((out, *grads), oracle.attention(q, k, v, lens, lens, scale=scale, dout=dout))


# ---- norm + rotation of many rows -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('M,H,G,D', [(30011, 13, 5, 64), (9001, 33, 7, 128), (60007, 16, 3, 64), (150001, 1, 6, 64)])
def test_norm_rope_of_many_rows(ops, eng, dtype, M, H, G, D):
    """Several heads a thread (a count that does not divide the heads), a launch of as many blocks as there may be, each of them over many rows."""
    assert M * (H + G) * (D // 16) > 1 << 20
    lib = _lib.load()
    assert lib.some_train_qk_norm_rope_bytes(None, M, H, G, D) == 1536 * D * 4
    fused = _normal(81, M, H + 2 * G, D, dtype=dtype, scale=1.7)
    q, k = fused[:, :H], fused[:, H:H + G]
    gq, gk = 1 + _normal(83, D, scale=0.3), 1 + _normal(84, D, scale=0.3)
    pos = torch.randint(-50, 3000000, (M,), device='cuda', generator=torch.Generator(device='cuda').manual_seed(85))
    dq, dk = _normal(86, M, H, D, dtype=dtype), _normal(87, M, G, D, dtype=dtype)
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
