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
