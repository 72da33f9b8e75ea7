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


# ------------------------------------------------------------------ incoming gradients of any size
def _exact_gradients(q, k, v, do, n, causal):
    """Of sequences of n rows each, in 64 bits."""
    T, hq, d = q.shape
    G, sc = hq // k.shape[1], 1 / math.sqrt(d)
    out = [torch.zeros_like(t, dtype=torch.float64) for t in (q, k, v)]
    hidden = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1) if causal else None
    for at in range(0, T, n):
        r = slice(at, at + n)
        for h in range(hq):
            qq, kk, vv, gg = (t.detach().double() for t in (q[r, h], k[r, h // G], v[r, h // G], do[r, h]))
            s = qq @ kk.T * sc
            p = torch.softmax(s if hidden is None else s.masked_fill_(hidden, -math.inf), 1)
            del s
            ds = gg @ vv.T
            ds = ds.sub_((p * ds).sum(1, keepdim=True)).mul_(p).mul_(sc)
            out[0][r, h] = ds @ kk
            out[1][r, h // G] += ds.T @ qq
            out[2][r, h // G] += p.T @ gg
    return out


@pytest.mark.parametrize("n,reps,do_scale,q_scale,k_scale,v_scale", [
    (12000, 1, 1e-2, 1, 1, 1), (12000, 1, 1e-3, 1, 1, 1),  # dS about 1 / n: below what fp16 holds well
    (40, 30, 2.0 ** -15, 1 / 16, 16, 1), (40, 30, 2.0 ** -15, 16, 1 / 16, 1),  # the same in short sequences
    (300, 2, 2.0 ** 12, 1 / 16, 1 / 16, 4), (50, 9, 2.0 ** 12, 1 / 16, 1 / 16, 4),  # dS past fp16's largest
])
@pytest.mark.parametrize("hq,hkv", [(2, 1), (2, 2)])  # the group's heads shared out, and not
@pytest.mark.parametrize("d,causal", [(64, True), (128, False)])
def test_fp16_gradients_of_small_and_large_incoming_gradients(n, reps, do_scale, q_scale, k_scale, v_scale, hq, hkv, d,
                                                              causal):
    """P, dS and the result are rounded once each, whatever the size of dS: three errors of h / sqrt(3)."""
    g = torch.Generator(device="cuda").manual_seed(n + d)
    T, f16 = n * reps, torch.float16
    q, k, v, do = (_rnd(g, T, x, d, dtype=f16, scale=s)
                   for x, s in ((hq, q_scale), (hkv, k_scale), (hkv, v_scale), (hq, do_scale)))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(attention_packed(*leaves, PackedBatch([n] * reps), causal=causal), leaves, do)
    h = HALF[f16]
    late = torch.arange(T, device="cuda") % n >= n // 2  # rows of many keys, which early rows would hide
    for name, got, want in zip(("dq", "dk", "dv"), grads, _exact_gradients(q, k, v, do, n, causal)):
        assert got.isfinite().all(), name
        for rows in (late, ~late):
            err, norm = (got[rows].double() - want[rows]).norm().item(), want[rows].norm().item()
            allowed = 1.5 * math.sqrt((h * norm) ** 2 + want[rows].numel() * STEP[f16] ** 2 / 12)
            assert err <= allowed, (name, err, norm, allowed)


# ------------------------------------------------------------------ one chunk of a prefix, nothing to join
@pytest.mark.parametrize("B,h", [(130, 128), (2, 256)])  # tiles that 128 rows share; a wave's own tiles
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_single_chunk_of_a_prefix_is_written_without_a_join(B, h, dtype):
    g = torch.Generator(device="cuda").manual_seed(B)
    P, d = 600, 64
    q, k, v = (_rnd(g, *s, dtype=dtype) for s in ((B, h, d), (h, P, d), (h, P, d)))
    own = torch.zeros(B, h, 0, d, device="cuda", dtype=dtype)
    att = dec.PrefixDecodeAttention(B, h, h, d, 0, P, "cuda", dtype=dtype)
    assert att.words == 0
    o = att(q, k, v, own, own, torch.zeros(B, device="cuda", dtype=torch.int32)).double()
    p = torch.softmax(torch.matmul(q.double().transpose(0, 1), k.double().transpose(1, 2).contiguous()) / 8, -1)
    want, mass = (torch.matmul(p, x).transpose(0, 1) for x in (v.double(), v.double().abs()))
    hf = HALF[dtype]
    assert ((o - want).abs() <= hf * want.abs() + (hf + 2.0 ** -14) * mass + STEP[dtype]).all()


def test_sequences_without_keys_are_written_where_chunks_are_joined():
    """Own chunks outside the one-workgroup form: whatever the cache's length, an empty sequence's zeros come from the
    join."""
    g = torch.Generator(device="cuda").manual_seed(1)
    for smax in (513, 700, 1025):
        q, kc, vc = (_rnd(g, *s, dtype=torch.bfloat16) for s in ((3, 4, 64), (3, 2, smax, 64), (3, 2, smax, 64)))
        none = kc[0, :, :0]
        for B in (3, 1):
            att = dec.PrefixDecodeAttention(B, 4, 2, 64, smax, 0, "cuda")
            o = att(q[:B], none, none, kc[:B], vc[:B], torch.tensor([0, 1, 0][:B], dtype=torch.int32, device="cuda"))
            assert not o[0].any() and not o[2:].any()
            assert B == 1 or torch.equal(o[1], vc[1, :, 0].repeat_interleave(2, 0))


# ------------------------------------------------------------------ D from the unrounded output
@pytest.mark.parametrize("n,reps", [(65, 8), (130, 4), (300, 2)])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (128, torch.float16)])
def test_gradients_take_d_from_the_unrounded_output(n, reps, d, dtype):
    """Values and keys around a common mean: an error of D_i moves all dS of the row one way, where the errors of the
    roundings of P and dS cancel.  The kernel's dQ and dK are within 1.5 times those roundings' root mean square; with
    D = dO . round(o) they would not be, which is computed beside it.  Not causal: every row has n keys."""
    g = torch.Generator(device="cuda").manual_seed(n + d)
    hq, hkv, T, sc, h = 2, 1, n * reps, 1 / math.sqrt(d), HALF[dtype]
    q, do = _rnd(g, T, hq, d, dtype=dtype), _rnd(g, T, hq, d, dtype=dtype)
    k, v = ((torch.randn(T, hkv, d, device="cuda", generator=g) + m).to(dtype) for m in (2, 4))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dq, dk, _ = torch.autograd.grad(attention_packed(*leaves, PackedBatch([n] * reps), causal=False), leaves, do)
    shape = [torch.zeros(T, x, d, device="cuda", dtype=torch.float64) for x in (hq, hkv)]
    want, off = [t.clone() for t in shape], [t.clone() for t in shape]  # the gradient; what D = dO . round(o) would add
    square = [torch.zeros_like(t[..., 0]) for t in shape]  # expected squared error of a row
    for at in range(0, T, n):
        r = slice(at, at + n)
        for hd in range(hq):
            qq, kk, vv, gg = (t.detach().double() for t in (q[r, hd], k[r, 0], v[r, 0], do[r, hd]))
            p = torch.softmax(qq @ kk.T * sc, 1)
            dp, o = gg @ vv.T, p @ vv
            ds = p * (dp - (gg * o).sum(1, keepdim=True))
            moved = p * -(gg * (o.to(dtype).double() - o)).sum(1, keepdim=True)
            want[0][r, hd], off[0][r, hd] = ds @ kk * sc, moved @ kk * sc
            want[1][r, 0] += ds.T @ qq * sc
            off[1][r, 0] += moved.T @ qq * sc
            # squared errors of D: P's roundings, that of o's low part, and fp32's (2^-20 of the summed magnitudes)
            d2 = h * h / 3 * (p * dp).pow(2).sum(1) + h ** 4 / 3 * (gg * o).pow(2).sum(1)
            d2 = d2 + (2.0 ** -20 * (gg.abs() * vv.abs().amax(0)).sum(1)) ** 2
            square[0][r, hd] = (h * h / 3 * (ds * ds) @ kk.pow(2).sum(1) + d2 * (p @ kk).pow(2).sum(1)) * sc * sc
            square[1][r, 0] += (h * h / 3 * (ds * ds).T @ qq.pow(2).sum(1) + (p * p).T @ (d2 * qq.pow(2).sum(1))) * sc * sc
    for name, got, val, var, sq in zip(("dq", "dk"), (dq, dk), want, off, square):
        allowed = 1.5 * math.sqrt(sq.sum().item() + h * h / 3 * val.pow(2).sum().item() + val.numel() * STEP[dtype] ** 2 / 12)
        err = (got.double() - val).norm().item()
        assert err <= allowed < var.norm().item(), (name, err, allowed, var.norm().item())


# ------------------------------------------------------------------ a plan dropped under a waiting launch
def test_a_dropped_plan_is_not_handed_out_before_its_launch_has_run():
    """The side stream is held back by a bounded spin, so the job table is certainly still to be read when the batch
    goes and tensors of its size are made on the main stream."""
    g = torch.Generator(device="cuda").manual_seed(14)
    lengths = [3000, 2000, 1]
    q, k, v = (_rnd(g, sum(lengths), x, 64, dtype=torch.bfloat16) for x in (16, 4, 4))
    want = attention_packed(q, k, v, PackedBatch(lengths))
    side, main = torch.cuda.Stream(), torch.cuda.current_stream()
    with torch.cuda.stream(side):
        attention_packed(q, k, v, PackedBatch(lengths))  # the stream's first call is not the one that counts
    torch.cuda.synchronize()
    batch = PackedBatch(lengths)
    at, slots = batch.jobs.data_ptr(), batch.jobs.shape[0]
    side.wait_stream(main)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got = attention_packed(q, k, v, batch)
    del batch
    other = [torch.zeros(slots, 4, dtype=torch.int32, device="cuda") for _ in range(8)]
    assert not side.query()  # the launch is still to come
    assert at not in [t.data_ptr() for t in other]
    main.wait_stream(side)
    assert torch.equal(got, want)


# ------------------------------------------------------------------ scores past 2^24
@pytest.mark.parametrize("scale", [300.0, 3000.0, 6000.0])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.float16), (128, torch.bfloat16)])
def test_huge_scores_choose_their_key(scale, d, dtype):
    """Scores of 1e5 to 1e8: an fp32 exponent is off by up to several units there, which must not carry a lifted
    probability past fp16's largest value.  Rows whose best key leads by far (2^-18 of the scores' size and 60 units,
    well past every rounding) give its value; gradients are finite."""
    g = torch.Generator(device="cuda").manual_seed(d)
    n, hq, hkv = 700, 4, 2
    q, k = _rnd(g, n, hq, d, dtype=dtype, scale=scale), _rnd(g, n, hkv, d, dtype=dtype, scale=scale)
    k[:200] *= 0.1  # maxima that rise
    v, do = _rnd(g, n, hkv, d, dtype=dtype), _rnd(g, n, hq, d, dtype=dtype)
    batch = PackedBatch([n])

    def check(o, keys, vals, seen=None):
        for h in range(hq):
            s = q[:, h].double() @ keys[h // 2].double().T / math.sqrt(d)
            s = s if seen is None else s.masked_fill(~seen, -math.inf)
            best = s.topk(2, 1)
            led = best.values[:, 0] - best.values[:, 1] > 60 + 2.0 ** -18 * s.masked_fill(s == -math.inf, 0).abs().amax(1)
            assert led.sum() > n // 2
            want = vals[h // 2][best.indices[led, 0]].double()
            # the one probability left is 2^x for some x <= 4, rounded once and divided by its unrounded self: 1 + h at
            # most; then the result's own rounding, and 2^-20 for fp32's
            assert ((o[led, h].double() - want).abs() <= (2 * HALF[dtype] + HALF[dtype] ** 2 + 2.0 ** -20) * want.abs()
                    + STEP[dtype]).all()

    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    for causal in (True, False):
        o = attention_packed(*leaves, batch, causal=causal)
        assert all(t.isfinite().all() for t in (o, *torch.autograd.grad(o, leaves, do)))
        if not causal:
            check(o.detach(), k.detach().transpose(0, 1), v.detach().transpose(0, 1))
    with torch.no_grad():
        # each row as the single token of a sequence behind the others' keys
        pk, pv = k.transpose(0, 1).contiguous(), v.transpose(0, 1).contiguous()
        own = torch.zeros(n, hkv, 8, d, device="cuda", dtype=dtype)
        att = dec.PrefixDecodeAttention(n, hq, hkv, d, 8, n, "cuda", dtype=dtype)
        check(att(q, pk, pv, own, own, torch.zeros(n, dtype=torch.int32, device="cuda")), pk, pv)
        few = dec.PrefixDecodeAttention(8, hq, hkv, d, 8, n, "cuda", dtype=dtype)
        o = torch.cat([few(q[i:i + 8].contiguous(), pk, pv, own[:8], own[:8], torch.zeros(8, dtype=torch.int32, device="cuda"))
                       for i in range(0, n - 4, 8)] + [torch.zeros_like(q[:n % 8])])
        keep = n - n % 8
        q, n = q[:keep], keep
        check(o[:keep], pk, pv)
