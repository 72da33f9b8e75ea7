"""Packed and prefix attention where a 16-bit type's range, or a rounding that
must not be there, decides: far keys, small and large incoming gradients, D
from the unrounded output.

h = eps / 2 is the largest relative error of one rounding; over many elements
its root mean square is at most h / sqrt(3).  Errors of independent roundings
add up in squares, so the checks below compare norms of many elements with
that root mean square and allow 1.5 times it.  fp16 outputs are also off by up
to half a step of 2^-24, a root mean square of 2^-24 / sqrt(12).
"""
import math

import pytest
import torch

from kgwe.ops import attention_packed
from kgwe.ops import decode as dec
from kgwe.ops.packed import PackedBatch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
STEP = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24}


def _rnd(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


# ------------------------------------------------------------------ far keys
def _far_keys(g, P, d, dtype):
    """Keys and values [1, P, d] of which the middle key outscores all others by 26 bits of probability and has a value
    of zero: the output is what the others add up to, about P 2^-26."""
    k, v = torch.zeros(1, P, d, device="cuda"), torch.rand(1, P, d, device="cuda", generator=g) + 0.5
    k[0, P // 2, 0], v[0, P // 2] = math.sqrt(26 * math.log(2) * math.sqrt(d)), 0
    q = k[:, P // 2].clone()
    return q.to(dtype), k.to(dtype), v.to(dtype)


def _check_far(o, q, k, v):
    """o [rows, d] for one query.  Every probability is rounded once (h; 2^-14 covers fp32's own roundings, as exponents
    of 26 carry 2^-18 into 2^x) and the result once; where fp16 holds a probability of 2^-26 of the row's largest, the
    largest is at least 2^11 and its step 2^-24: 2^-36 of the largest each."""
    p = torch.softmax(q.double() @ k[0].double().T / math.sqrt(k.shape[2]), 1)
    h = HALF[o.dtype]
    want, mass = p @ v[0].double(), p @ v[0].double()
    tol = h * want + (h + 2.0 ** -14) * mass + (STEP[o.dtype] * 2.0 ** -12 * v[0].double().sum(0))
    assert ((o.double() - want).abs() <= tol).all(), ((o.double() - want).abs() / want).max().item()


@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.float16), (128, torch.bfloat16)])
def test_many_far_keys_keep_their_weight(d, dtype):
    g = torch.Generator(device="cuda").manual_seed(d)
    P = 65536
    q, k, v = _far_keys(g, P, d, dtype)
    with torch.no_grad():
        # behind a prefix, its length alone; two halves per workgroup, and workgroups enough for one
        for n in (3, 20000):
            zero = torch.zeros(n, 1, d, device="cuda", dtype=dtype)
            o = attention_packed(q[:, None].expand(n, 1, d), zero, zero, PackedBatch([1] * n), prefix=(k, v))
            # a row's own key is one more far key, of value 0
            kk, vv = torch.cat([k, zero[:1, 0][None]], 1), torch.cat([v, zero[:1, 0][None]], 1)
            _check_far(o[:, 0], q, kk, vv)
        # as a sequence's own keys
        o = attention_packed(q.expand(P, 1, d).contiguous(), k[0, :, None], v[0, :, None], PackedBatch([P]), causal=False)
        _check_far(o[::4096, 0], q, k, v)
        # single tokens: at most 32 rows (a wave's own tiles), and tiles that 128 rows share
        for B in (2, 100):
            own = torch.zeros(B, 1, 300, d, device="cuda", dtype=dtype)
            att = dec.PrefixDecodeAttention(B, 1, 1, d, 300, P, "cuda", dtype=dtype)
            lens = torch.zeros(B, dtype=torch.int32, device="cuda")
            _check_far(att(q.expand(B, 1, d).contiguous(), k, v, own, own, lens)[:, 0], q, k, v)
