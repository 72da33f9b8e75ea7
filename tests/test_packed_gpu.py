"""The packed-batch kernels on a GPU against plain formulas in 64 bits.

Tolerances count roundings.  h = eps / 2 of the 16-bit type is the largest
relative error of one rounding to it.  Attention rounds P (and dS) once per
element and the result once; everything else is fp32, for which 2^-14 of the
summed magnitudes is allowed (exponents of a few tens of units carry about
2^-17 of relative error into 2^x, sums of at most a few thousand terms about
2^-14).  fp16 holds values below 2^-14 with an absolute step, so a probability
may be off by 2^-25 there (the row's largest is at least 1 before the division).
"""
import math

import pytest
import torch

from kgwe.ops import attention_packed, norm_rope_qkv
from kgwe.ops import decode as dec
from kgwe.ops import reference as ref
from kgwe.ops.packed import PackedBatch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
SLOP = 2.0 ** -14


def _rnd(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(dtype)


def _within(got, want, tol, what):
    assert got.isfinite().all(), what
    excess = (got.double() - want).abs() - tol
    assert excess.max().item() <= 0, (what, excess.max().item(), tol.max().item())


# ------------------------------------------------------------------ the plan
@pytest.mark.parametrize("lengths,total", [
    ([3, 0, 5], 10), ([], 3), ([0], 1), ([129, 1, 128, 127, 0, 300], 700), ([1] * 1500, 1500), ([70000], 70001),
    ([5, 6000, 1, 0, 2048] * 30, 30 * 8054 + 9)])
def test_plan_tables(lengths, total):
    host = PackedBatch(lengths, total=total, device="cpu")
    for batch in (PackedBatch(lengths, total=total),
                  PackedBatch(torch.tensor(lengths, dtype=torch.int32, device="cuda"), total=total)):
        for name in ("cu", "positions", "seq_ids", "last_rows"):
            assert torch.equal(getattr(batch, name).cpu(), getattr(host, name)), name
        jobs = [tuple(j) for j in batch.jobs.tolist() if j[1] > 0]
        full = [*lengths, total - sum(lengths)]
        assert sorted(jobs) == sorted((sum(full[:s]), n, b, n if s < len(lengths) else 0)
                                      for s, n in enumerate(full) for b in range((n + 127) // 128))
        sweep = [-1 if keys == 0 else min(b, 2046) for _, _, b, keys in jobs]
        assert sweep == sorted(sweep, reverse=True)  # longest first, padding last


def test_plan_of_lengths_that_do_not_fit_stays_inside():
    lengths = torch.tensor([5, -7, 2**31 - 1, 2**31 - 1, 4], dtype=torch.int32, device="cuda")
    batch = PackedBatch(lengths, total=300)
    assert batch.cu.tolist() == [0, 5, 5, 300, 300, 300, 300]
    assert sorted(j for j in batch.jobs.tolist() if j[1] > 0) == [[0, 5, 0, 5], *([5, 295, b, 295] for b in range(3))]
    with pytest.raises(ValueError):
        PackedBatch(lengths)


# ------------------------------------------------------------------ attention
def _exact_attention(q, k, v, lengths, causal, prefix=None, do=None):
    """Formulas in 64 bits; per output (value, the magnitudes a tolerance needs)."""
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    h, tiny = HALF[q.dtype], TINY[q.dtype]
    q, k, v = q.detach().double(), k.detach().double(), v.detach().double()
    G, sc = hq // hkv, 1.0 / math.sqrt(d)
    o, to = torch.zeros_like(q), torch.zeros_like(q)
    out = {n: (torch.zeros_like(t), torch.zeros_like(t)) for n, t in (("dq", q), ("dk", k), ("dv", v))}
    at = 0
    for n in lengths:
        r = slice(at, at + n)
        at += n
        if n == 0:
            continue
        i = torch.arange(n, device=q.device)
        for hd in range(hq):
            j = hd // G
            kk, vv = k[r, j], v[r, j]
            seen = i[:, None] >= i[None] if causal else torch.ones(n, n, dtype=torch.bool, device=q.device)
            if prefix is not None:
                kk, vv = torch.cat([prefix[0][j].double(), kk]), torch.cat([prefix[1][j].double(), vv])
                seen = torch.cat([torch.ones(n, len(kk) - n, dtype=torch.bool, device=q.device), seen], 1)
            p = torch.softmax((q[r, hd] @ kk.T * sc).masked_fill(~seen, -math.inf), 1)
            o[r, hd] = p @ vv
            mag = p @ vv.abs() + 0.0
            to[r, hd] = h * o[r, hd].abs() + (h + SLOP) * mag + tiny * (1 + len(kk) * vv.abs().max())
            if do is None:
                continue
            g = do[r, hd].double()
            dp, delta = g @ vv.T, (g * o[r, hd]).sum(1, keepdim=True)
            ds = p * (dp - delta)
            # dS: its own rounding, and D from the rounded output of the forward
            edelta = (g.abs() * to[r, hd]).sum(1, keepdim=True)
            eds = h * ds.abs() + p * edelta + SLOP * p * (g.abs() @ vv.abs().T + (g * o[r, hd]).abs().sum(1, keepdim=True))
            eds = eds + tiny * seen
            ep = ((h + SLOP) * p + tiny) * seen
            for name, val, err, mags in (("dq", ds @ kk * sc, eds @ kk.abs() * sc, ds.abs() @ kk.abs() * sc),):
                out[name][0][r, hd] += val
                out[name][1][r, hd] += err + SLOP * mags
            out["dk"][0][r, j] += ds.T @ q[r, hd] * sc
            out["dk"][1][r, j] += (eds + SLOP * ds.abs()).T @ q[r, hd].abs() * sc
            out["dv"][0][r, j] += p.T @ g
            out["dv"][1][r, j] += ep.T @ g.abs()
    if do is None:
        return o, to
    grads = {n: (val, err + h * val.abs() + tiny) for n, (val, err) in out.items()}
    return o, to, grads


SHAPES = [
    ([1], 0, 4, 4, 64, True), ([5, 0, 1, 70], 3, 4, 2, 64, True), ([64, 65, 63, 128, 129, 127], 0, 8, 2, 128, True),
    ([300, 2, 511], 130, 8, 1, 64, False), ([257, 40], 1, 6, 2, 128, False), ([1000, 1], 0, 5, 5, 128, True),
    ([31, 32, 33] * 5, 0, 16, 2, 64, True), ([0, 0], 5, 4, 2, 128, True), ([200], 300, 3, 1, 64, True),
]


@pytest.mark.parametrize("lengths,pad,hq,hkv,d,causal", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_packed_attention_and_gradient(lengths, pad, hq, hkv, d, causal, dtype):
    g = torch.Generator(device="cuda").manual_seed(len(lengths) + d)
    T = sum(lengths) + pad
    # slices of one fused projection: strided views, odd row strides
    qkv = _rnd(g, T, (hq + 2 * hkv + 1) * d, dtype=dtype).view(T, -1, d)
    qkv[sum(lengths):] = float("nan")  # padding is never looked at
    q, k, v = (qkv[:, a:b].detach().requires_grad_(True)
               for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    do = _rnd(g, T, hq, d, dtype=dtype)
    do[sum(lengths):] = float("nan")
    o = attention_packed(q, k, v, PackedBatch(lengths, total=T), causal=causal)
    grads = torch.autograd.grad(o, (q, k, v), do)
    want, tol, exact = _exact_attention(q, k, v, lengths, causal, do=do)
    _within(o, want, tol, "o")
    for name, got in zip(("dq", "dk", "dv"), grads):
        _within(got, *exact[name], name)


@pytest.mark.parametrize("hq,hkv", [(32, 16), (21, 3)])  # no join of dK / dV; four parts, the last of one head
@pytest.mark.parametrize("d,dtype,causal", [(128, torch.bfloat16, True), (128, torch.float16, False),
                                            (64, torch.float16, True)])
def test_packed_attention_and_gradient_of_many_blocks(hq, hkv, d, dtype, causal):
    """Workgroups enough for every CU: at D = 128 the form with one V buffer."""
    g = torch.Generator(device="cuda").manual_seed(hq + d)
    lengths, pad = [20] * 30 + [300, 0, 150] + [1, 33] * 14, 7
    T = sum(lengths) + pad
    q, k, v = (_rnd(g, T, h, d, dtype=dtype).requires_grad_(True) for h in (hq, hkv, hkv))
    do = _rnd(g, T, hq, d, dtype=dtype)
    o = attention_packed(q, k, v, PackedBatch(lengths, total=T), causal=causal)
    grads = torch.autograd.grad(o, (q, k, v), do)
    want, tol, exact = _exact_attention(q, k, v, lengths, causal, do=do)
    _within(o, want, tol, "o")
    for name, got in zip(("dq", "dk", "dv"), grads):
        _within(got, *exact[name], name)
    prefix = _rnd(g, hkv, 150, d, dtype=dtype), _rnd(g, hkv, 150, d, dtype=dtype)
    with torch.no_grad():
        o = attention_packed(q, k, v, PackedBatch(lengths, total=T), causal=causal, prefix=prefix)
    _within(o, *_exact_attention(q, k, v, lengths, causal, prefix=prefix), "o")


@pytest.mark.parametrize("P", [1, 63, 64, 200])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_behind_a_prefix(P, d, dtype, causal):
    g = torch.Generator(device="cuda").manual_seed(P)
    lengths, pad, hq, hkv = [1, 130, 0, 64, 7], 2, 8, 2
    T = sum(lengths) + pad
    q, k, v = _rnd(g, T, hq, d, dtype=dtype), _rnd(g, T, hkv, d, dtype=dtype), _rnd(g, T, hkv, d, dtype=dtype)
    # the prefix lies in a longer cache, and what follows it there is garbage
    cache = torch.full((2, hkv, P + 9, d), float("nan"), device="cuda", dtype=dtype)
    cache[:, :, :P] = _rnd(g, 2, hkv, P, d, dtype=dtype)
    pk, pv = cache[0, :, :P], cache[1, :, :P]
    o = attention_packed(q, k, v, PackedBatch(lengths, total=T), causal=causal, prefix=(pk, pv))
    _within(o, *_exact_attention(q, k, v, lengths, causal, prefix=(pk, pv)), "o")
    none = attention_packed(q, k, v, PackedBatch(lengths, total=T), causal=causal, prefix=(pk[:, :0], pv[:, :0]))
    assert torch.equal(none, attention_packed(q, k, v, PackedBatch(lengths, total=T), causal=causal))


@pytest.mark.parametrize("d", [64, 128])
def test_broadcast_rows_and_single_rows(d):
    """Inputs whose rows are one row (stride 0), overlap, or lie alone in a row of odd width."""
    g = torch.Generator(device="cuda").manual_seed(d)
    lengths, hq, hkv = [3, 130], 4, 2
    T, batch = sum(lengths), PackedBatch(lengths)
    q1, k1, v1 = _rnd(g, 1, hq, d), _rnd(g, 1, hkv, d), _rnd(g, T, 1, d)
    do = _rnd(g, T, hq, d)
    leaves = [t.requires_grad_(True) for t in (q1, k1, v1)]

    def call(make):
        x = [make(t.expand(T, h, d)) for t, h in zip(leaves, (hq, hkv, hkv))]
        o = attention_packed(*x, batch)
        return o, *torch.autograd.grad(o, leaves, do)

    for a, b in zip(call(lambda t: t), call(lambda t: t.contiguous())):
        assert torch.equal(a, b)
    # a prefix of one row repeated, in both calls that take one
    row, P = _rnd(g, hkv, 1, d), 70
    pk = pv = row.expand(hkv, P, d)
    with torch.no_grad():
        q, k, v = (t.detach().expand(T, h, d).contiguous() for t, h in zip(leaves, (hq, hkv, hkv)))
        assert torch.equal(attention_packed(q, k, v, batch, prefix=(pk, pv)),
                           attention_packed(q, k, v, batch, prefix=(pk.contiguous(), pv.contiguous())))
        kc, vc = _rnd(g, T, hkv, 16, d), _rnd(g, T, hkv, 16, d)
        lens = torch.arange(T, device="cuda", dtype=torch.int32) % 17
        for B in (3, T):
            att = dec.PrefixDecodeAttention(B, hq, hkv, d, 16, P, "cuda")
            args = kc[:B], vc[:B], lens[:B]
            assert torch.equal(att(q[:B], pk, pv, *args), att(q[:B], pk.contiguous(), pv.contiguous(), *args))
        # one row of a wider, odd buffer
        wide = _rnd(g, 2, (hq + 2 * hkv) * d + 3)
        one = wide[:1, :(hq + 2 * hkv) * d]
        cos, sin = torch.rand(2, 8, d // 2, device="cuda").unbind()
        pos = torch.tensor([5], dtype=torch.int32, device="cuda")
        got = norm_rope_qkv(one, cos, sin, pos, hq, hkv, d)
        for a, b in zip(got, norm_rope_qkv(one.clone(), cos, sin, pos, hq, hkv, d)):
            assert torch.equal(a, b)
        x = [one.view(1, -1, d)[:, i:i + h] for i, h in ((0, hq), (hq, hkv), (hq + hkv, hkv))]
        assert torch.equal(attention_packed(*x, PackedBatch([1])), x[2].repeat_interleave(hq // hkv, 1))


def test_neighbours_do_not_enter():
    """A sequence's outputs and gradients are its own: the same bits whatever the others hold, NaN included."""
    g = torch.Generator(device="cuda").manual_seed(5)
    lengths, hq, hkv, d = [70, 100, 90], 4, 2, 128
    T = sum(lengths)
    batch = PackedBatch(lengths)
    x = [_rnd(g, T, h, d) for h in (hq, hkv, hkv, hq)]

    def go(parts):
        q, k, v = (t.clone().requires_grad_(True) for t in parts[:3])
        o = attention_packed(q, k, v, batch)
        return [t[70:170] for t in (o, *torch.autograd.grad(o, (q, k, v), parts[3]))]

    want = go(x)
    y = [t.clone() for t in x]
    for t in y:
        t[:70] = float("nan")
        t[170:] = float("inf")
    for a, b in zip(go(y), want):
        assert torch.equal(a, b)


def test_large_scores_and_growing_maximum():
    g = torch.Generator(device="cuda").manual_seed(6)
    n, hq, hkv, d = 700, 4, 1, 64
    q, v = _rnd(g, n, hq, d, scale=3.0), _rnd(g, n, hkv, d)
    k = (torch.randn(n, hkv, d, device="cuda", generator=g) * torch.linspace(0.1, 6, n, device="cuda")[:, None, None]).bfloat16()
    o = attention_packed(q, k, v, PackedBatch([n]))
    _within(o, *_exact_attention(q, k, v, [n], True), "o")


@pytest.mark.parametrize("lengths,pad,P,hq,hkv,causal", [
    ([700], 0, 0, 4, 1, True), ([1111], 3, 0, 3, 3, False), ([641, 640], 0, 0, 6, 2, True),
    ([1, 130, 0, 64, 33], 2, 700, 8, 2, True), ([20], 0, 641, 4, 4, False), ([90], 0, 1000, 2, 1, True),
])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16), (128, torch.bfloat16)])
def test_long_sweeps_of_few_workgroups(lengths, pad, P, hq, hkv, causal, d, dtype):
    """Sweeps that two halves of a workgroup share: odd and even tile counts, rows that see one half's tiles only."""
    g = torch.Generator(device="cuda").manual_seed(P + hq)
    T = sum(lengths) + pad
    q, k, v = (_rnd(g, T, h, d, dtype=dtype) for h in (hq, hkv, hkv))
    prefix = (_rnd(g, hkv, P, d, dtype=dtype), _rnd(g, hkv, P, d, dtype=dtype)) if P else None
    o = attention_packed(q, k, v, PackedBatch(lengths, total=T), causal=causal, prefix=prefix)
    _within(o, *_exact_attention(q, k, v, lengths, causal, prefix=prefix), "o")
    if P == 0:
        do = _rnd(g, T, hq, d, dtype=dtype)
        for t in (q, k, v):
            t.requires_grad_(True)
        o = attention_packed(q, k, v, PackedBatch(lengths, total=T), causal=causal)
        grads = torch.autograd.grad(o, (q, k, v), do)
        exact = _exact_attention(q, k, v, lengths, causal, do=do)[2]
        for name, got in zip(("dq", "dk", "dv"), grads):
            _within(got, *exact[name], name)


@pytest.mark.parametrize("n", [2, 3, 17, 64])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("causal", [True, False])
def test_gradients_of_short_sequences_are_rounded_once(n, d, dtype, causal):
    """dQ and dK of sequences of up to 64 rows: dS is two 16-bit values (h^2 of it is lost, or half an fp16 step) and D the sum of P dP in
    fp32, so but for fp32's own roundings the error is that of the result, h."""
    g = torch.Generator(device="cuda").manual_seed(n)
    hq, hkv, reps = 6, 3, 5
    lengths, h, tiny, sc = [n] * reps, HALF[dtype], TINY[dtype], 1 / math.sqrt(d)
    q, k, v, do = (_rnd(g, n * reps, x, d, dtype=dtype) for x in (hq, hkv, hkv, hq))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dq, dk, _ = torch.autograd.grad(attention_packed(*leaves, PackedBatch(lengths), causal=causal), leaves, do)
    seen = torch.ones(n, n, device="cuda", dtype=torch.bool).tril() if causal else torch.ones(
        n, n, device="cuda", dtype=torch.bool)
    want = [torch.zeros_like(t, dtype=torch.float64) for t in (dq, dk)]
    tol = [torch.zeros_like(t) for t in want]
    for i in range(reps):
        r = slice(i * n, i * n + n)
        for hd in range(hq):
            j = hd // (hq // hkv)
            qq, kk, vv, gg = (t.detach().double() for t in (q[r, hd], k[r, j], v[r, j], do[r, hd]))
            p = torch.softmax((qq @ kk.T * sc).masked_fill(~seen, -math.inf), 1)
            dp, mag = gg @ vv.T, gg.abs() @ vv.abs().T
            ds = p * (dp - (p * dp).sum(1, keepdim=True))
            eds = (h * h + SLOP) * ds.abs() + SLOP * p * (mag + (p * mag).sum(1, keepdim=True)) + tiny * seen
            want[0][r, hd], tol[0][r, hd] = ds @ kk * sc, (eds + SLOP * ds.abs()) @ kk.abs() * sc
            want[1][r, j] += ds.T @ qq * sc
            tol[1][r, j] += (eds + SLOP * ds.abs()).T @ qq.abs() * sc
    for got, val, t, name in zip((dq, dk), want, tol, ("dq", "dk")):
        _within(got, val, t + h * val.abs() + tiny, name)


def test_gradient_matches_differences():
    g = torch.Generator(device="cuda").manual_seed(7)
    lengths, hq, hkv, d = [37, 80], 4, 2, 64
    T = sum(lengths)
    x = [_rnd(g, T, h, d, dtype=torch.float16) for h in (hq, hkv, hkv)]
    do = _rnd(g, T, hq, d, dtype=torch.float16)
    q, k, v = (t.clone().requires_grad_(True) for t in x)
    grads = torch.autograd.grad(attention_packed(q, k, v, PackedBatch(lengths)), (q, k, v), do)
    step = [torch.randn(t.shape, device="cuda", generator=g, dtype=torch.float64) for t in x]

    def value(s):  # the formula in 64 bits
        y = [t.double() + s * e for t, e in zip(x, step)]
        y = [t.to(torch.float64) for t in y]
        total, at = 0.0, 0
        for n in lengths:
            r = slice(at, at + n)
            at += n
            for h in range(hq):
                sc = y[0][r, h] @ y[1][r, h // 2].T / 8
                sc = sc.masked_fill(torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1), -math.inf)
                total = total + ((sc.softmax(1) @ y[2][r, h // 2]) * do[r, h].double()).sum()
        return total.item()

    diff = (value(1e-4) - value(-1e-4)) / 2e-4
    got = sum((a.double() * s).sum().item() for a, s in zip(grads, step))
    # every gradient element is off by a few roundings (2^-11) of its own size, with random signs
    size = sum((a.double() * s).pow(2).sum().item() for a, s in zip(grads, step)) ** 0.5
    assert abs(diff - got) < 8 * 2.0 ** -11 * size + 1e-5 * abs(diff), (diff, got, size)


def test_repeats_bit_for_bit_and_on_another_stream():
    g = torch.Generator(device="cuda").manual_seed(8)
    lengths, hq, hkv, d = [500, 3, 260], 8, 2, 64
    T = sum(lengths)
    batch = PackedBatch(lengths)
    q, k, v = (_rnd(g, T, h, d).requires_grad_(True) for h in (hq, hkv, hkv))
    do = _rnd(g, T, hq, d)

    def go():
        o = attention_packed(q, k, v, batch)
        return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))

    want = go()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = go()
    torch.cuda.current_stream().wait_stream(s)
    for a, b, c in zip(want, again, go()):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_a_batch_dropped_while_another_stream_uses_it():
    """The job table is marked as in use on the stream of the launch: memory handed out after the batch is
    gone does not come from under the kernel."""
    g = torch.Generator(device="cuda").manual_seed(14)
    lengths = [3000, 2000, 1]
    T = sum(lengths)
    q, k, v = (_rnd(g, T, h, 64) for h in (16, 4, 4))
    want = attention_packed(q, k, v, PackedBatch(lengths))
    s = torch.cuda.Stream()
    for _ in range(4):
        batch = PackedBatch(lengths)
        slots = batch.jobs.shape[0]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = attention_packed(q, k, v, batch)
        del batch
        other = [torch.zeros(slots, 4, dtype=torch.int32, device="cuda") for _ in range(8)]  # rows = 0 everywhere
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(got, want)
        del other


def test_far_rows_are_copied():
    """A row stride past the kernels' 32-bit tile offsets: a copy, not a refusal."""
    base = torch.zeros(5 * ((1 << 22) + 8), device="cuda", dtype=torch.bfloat16)
    q = base.as_strided((5, 2, 64), ((1 << 22) + 8, 64, 1))
    q.copy_(torch.randn(5, 2, 64, device="cuda"))
    b = PackedBatch([5])
    assert torch.equal(attention_packed(q, q, q, b), attention_packed(*[q.contiguous()] * 3, b))


def test_captured_with_its_plan_and_replayed():
    """The plan is built inside the capture from lengths on the GPU: a replay follows new lengths."""
    g = torch.Generator(device="cuda").manual_seed(9)
    T, hq, hkv, d = 400, 4, 2, 128
    q, k, v = (_rnd(g, T, h, d) for h in (hq, hkv, hkv))
    lengths = torch.tensor([100, 200, 50], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        attention_packed(q, k, v, PackedBatch(lengths, total=T))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = attention_packed(q, k, v, PackedBatch(lengths, total=T))
        for new in ([100, 200, 50], [1, 0, 399], [0, 0, 0], [400, 5, 5], [130, 130, 130]):
            lengths.copy_(torch.tensor(new, dtype=torch.int32))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, attention_packed(q, k, v, PackedBatch(lengths, total=T))), new


def test_gradients_captured_and_replayed():
    """Rotation, attention and both gradients in one graph; every replay gives the eager call's bits."""
    g = torch.Generator(device="cuda").manual_seed(10)
    T, hq, hkv, d = 300, 8, 2, 128
    x, w = _rnd(g, T, (hq + 2 * hkv) * d), [_rnd(g, d) for _ in range(2)]
    cos, sin = torch.rand(2, T, d // 2, device="cuda", generator=g).unbind()
    do, batch = _rnd(g, T, hq, d), PackedBatch([100, 3, 190], total=T)
    leaves = [t.requires_grad_(True) for t in (x, *w)]

    def call():
        q, k, v = norm_rope_qkv(x, cos, sin, batch.positions, hq, hkv, d, *w)
        o = attention_packed(q, k, v, batch)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call()
    for _ in range(4):
        with torch.no_grad():
            x.copy_(_rnd(g, *x.shape))
            do.copy_(_rnd(g, *do.shape))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, call()):
            assert torch.equal(a, b)


def test_packed_attention_gpu_refusals():
    b = PackedBatch([4])
    q = torch.zeros(4, 2, 64, device="cuda")
    with pytest.raises(ValueError):
        attention_packed(q, q, q, b)  # fp32
    q = torch.zeros(4, 2, 32, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        attention_packed(q, q, q, b)  # head_dim
    q = torch.zeros(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        attention_packed(q, q, q, PackedBatch([4], device="cpu"))
    assert attention_packed(q[:0], q[:0], q[:0], PackedBatch([], device="cuda")).shape == (0, 2, 64)


# ------------------------------------------------------------------ norm + rotation
def _exact_norm_rope(qkv, cos, sin, pos, hq, hkv, d, wq, wk, eps, offset, dy=None):
    """64-bit values and tolerances.  All arithmetic is fp32 with fewer than 32
    roundings per element before the one to 16 bits: 2^-19 of the magnitudes."""
    h = HALF[qkv.dtype]
    T = qkv.shape[0]
    at = pos.long() + offset
    live = ((pos >= 0) & (at < cos.shape[0]))[:, None, None]
    at = at.clamp(0, cos.shape[0] - 1)
    x = qkv.detach().double().view(T, -1, d).masked_fill(~live, 0.0)
    c, s = cos[at].double()[:, None], sin[at].double()[:, None]
    tiny = 2 * TINY[qkv.dtype]
    parts, vals, tols = x.split((hq, hkv, hkv), 1), [], []

    def turn(t, sg):
        a, b = t.chunk(2, -1)
        return torch.cat([a * c - sg * b * s, b * c + sg * a * s], -1) * live

    def swap(t):
        a, b = t.abs().chunk(2, -1)
        return torch.cat([a + b, a + b], -1) * live

    for t, w in zip(parts[:2], (wq, wk)):
        n = t
        if w is not None:
            n = t / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + eps) * w.detach().double()
        vals.append(turn(n, 1))
        tols.append(h * vals[-1].abs() + 2.0 ** -19 * swap(n) + tiny)
    vals.append(parts[2])
    tols.append(torch.zeros_like(parts[2]))
    if dy is None:
        return vals, tols
    gvals, gtols, dws = [], [], []
    for t, w, y in zip(parts[:2], (wq, wk), dy):
        y = y.double().masked_fill(~live, 0.0)
        g, gm = turn(y, -1), swap(y)
        if w is None:
            gvals.append(g)
            gtols.append(h * g.abs() + 2.0 ** -19 * gm + tiny)
            continue
        w = w.detach().double()
        r = 1 / torch.sqrt(t.pow(2).mean(-1, keepdim=True) + eps)
        dx = r * (w * g - t * r * r * (w * g * t).mean(-1, keepdim=True))
        mag = r * ((w * gm).abs() + t.abs() * r * r * (w * gm * t).abs().mean(-1, keepdim=True))
        gvals.append(dx * live)
        gtols.append(h * dx.abs() + 2.0 ** -18 * mag + tiny)
        dw = (g * t * r).sum((0, 1))
        # sums of products: chains of at most a few hundred fp32 additions
        dws.append((dw, h * dw.abs() + 2.0 ** -16 * (gm * t * r).abs().sum((0, 1)) + tiny))
    gvals.append(dy[2].double().masked_fill(~live, 0.0))
    gtols.append(torch.zeros_like(gvals[-1]))
    return vals, tols, torch.cat(gvals, 1).view(T, -1), torch.cat(gtols, 1).view(T, -1), dws


@pytest.mark.parametrize("T,hq,hkv,d", [(1, 4, 1, 64), (7, 5, 5, 128), (130, 32, 8, 128), (33, 3, 1, 256),
                                        (64, 2, 2, 32), (1000, 12, 4, 64)])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_rope_and_gradient(T, hq, hkv, d, norm, dtype):
    g = torch.Generator(device="cuda").manual_seed(T)
    wide = _rnd(g, T, (hq + 2 * hkv) * d + 16, dtype=dtype, scale=1.5)
    qkv = wide[:, 8:-8].detach().requires_grad_(True)  # a strided view
    offset, eps = 3, 1e-5
    cos, sin = ref.rope_tables(T + 2, d, device="cuda")
    pos = torch.randint(0, T, (T,), device="cuda", generator=g, dtype=torch.int32)
    pos[T // 2] = T - 1  # its place is the table's end: p + offset is outside
    pos[0] = -1 if T > 1 else 0
    with torch.no_grad():
        wide[pos < 0] = float("nan")
    w = (1 + 0.3 * torch.randn(2, d, device="cuda", generator=g)).to(dtype)
    wq, wk = (w[0].clone().requires_grad_(True), w[1].clone().requires_grad_(True)) if norm else (None, None)
    dy = [_rnd(g, T, h, d, dtype=dtype) for h in (hq, hkv, hkv)]
    out = norm_rope_qkv(qkv, cos, sin, pos, hq, hkv, d, wq, wk, eps=eps, offset=offset)
    grads = torch.autograd.grad(out, (qkv, wq, wk) if norm else (qkv,), dy)
    vals, tols, dx, dxt, dws = _exact_norm_rope(qkv, cos, sin, pos, hq, hkv, d, wq, wk, eps, offset, dy)
    for name, got, want, tol in zip("qkv", out, vals, tols):
        _within(got, want, tol, name)
    _within(grads[0], dx, dxt, "dqkv")
    for name, got, (want, tol) in zip(("dwq", "dwk"), grads[1:], dws):
        _within(got, want, tol, name)
    again = torch.autograd.grad(norm_rope_qkv(qkv, cos, sin, pos, hq, hkv, d, wq, wk, eps=eps, offset=offset),
                                (qkv, wq, wk) if norm else (qkv,), dy)
    assert all(torch.equal(a, b) for a, b in zip(again, grads))


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_norm_rope_append(norm, d, dtype):
    g = torch.Generator(device="cuda").manual_seed(11)
    T, hq, hkv, smax, R, offset = 9, 6, 2, 20, 5, 4
    qkv = _rnd(g, T, (hq + 2 * hkv) * d, dtype=dtype)
    cos, sin = ref.rope_tables(smax + offset, d, device="cuda")
    pos = torch.tensor([0, 19, 20, -1, 5, 6, 7, 19, 0], dtype=torch.int32, device="cuda")
    rows = torch.tensor([0, 1, 2, 3, 4, 4, 5, -1, 4], dtype=torch.int32, device="cuda")
    w = (1 + 0.3 * torch.randn(2, d, device="cuda", generator=g)).to(dtype)
    wq, wk = (w[0], w[1]) if norm else (None, None)
    kc, vc = _rnd(g, R, hkv, smax, d, dtype=dtype), _rnd(g, R, hkv, smax, d, dtype=dtype)
    k0, v0 = kc.clone(), vc.clone()
    q, k, v = dec.norm_rope_append(qkv, pos, cos, sin, kc, vc, hq, hkv, d, wq, wk, offset=offset, rows=rows, keep_kv=True)
    for a, b in zip((q, k, v), norm_rope_qkv(qkv, cos, sin, pos, hq, hkv, d, wq, wk, offset=offset)):
        assert torch.equal(a, b)
    for t in range(T):
        r, p = int(rows[t]), int(pos[t])
        if 0 <= r < R and 0 <= p < smax:
            k0[r, :, p], v0[r, :, p] = k[t], v[t]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    # a decode step: row t is the cache's row t, q alone comes back
    step = dec.norm_rope_append(qkv[:R], pos[:R], cos, sin, kc, vc, hq, hkv, d, wq, wk, offset=offset)
    assert torch.equal(step, q[:R])


@pytest.mark.parametrize("norm", [True, False])
def test_norm_rope_of_a_rectangular_batch(norm):
    """A sequence length in the place of positions: the same bits as its table of positions."""
    g = torch.Generator(device="cuda").manual_seed(12)
    S, hq, hkv, d = 50, 4, 2, 64
    qkv = _rnd(g, 3 * S, (hq + 2 * hkv) * d).requires_grad_(True)
    cos, sin = ref.rope_tables(S, d, device="cuda")
    w = [(1 + 0.3 * torch.randn(d, device="cuda", generator=g)).bfloat16().requires_grad_(True) for _ in "qk"]
    dy = [_rnd(g, 3 * S, h, d) for h in (hq, hkv, hkv)]
    res = []
    for at in (S, PackedBatch([S] * 3).positions):
        out = norm_rope_qkv(qkv, cos, sin, at, hq, hkv, d, *(w if norm else ()))
        res.append([*out, *torch.autograd.grad(out, (qkv, *(w if norm else ())), dy)])
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_norm_rope_gpu_refusals():
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    cos, sin = ref.rope_tables(4, 48, device="cuda")
    with pytest.raises(ValueError):
        norm_rope_qkv(torch.zeros(2, 3 * 48, device="cuda", dtype=torch.bfloat16), cos, sin, pos, 1, 1, 48)
    cos, sin = ref.rope_tables(4, 64, device="cuda")
    with pytest.raises(ValueError):
        norm_rope_qkv(torch.zeros(2, 3 * 64, device="cuda"), cos, sin, pos, 1, 1, 64)
    with pytest.raises(ValueError):
        norm_rope_qkv(torch.zeros(2, 3 * 64, device="cuda", dtype=torch.bfloat16), cos, sin, pos.cpu(), 1, 1, 64)
    empty = norm_rope_qkv(torch.zeros(0, 3 * 64, device="cuda", dtype=torch.bfloat16), cos, sin, pos[:0], 1, 1, 64)
    assert [t.shape for t in empty] == [(0, 1, 64)] * 3


# ------------------------------------------------------------------ single tokens behind a shared prefix
def _exact_prefix(q, pk, pv, kc, vc, lens):
    h, tiny = HALF[q.dtype], TINY[q.dtype]
    out, tol = torch.zeros_like(q, dtype=torch.float64), torch.zeros_like(q, dtype=torch.float64)
    G = q.shape[1] // kc.shape[1]
    for b, n in enumerate(lens.tolist()):
        for j in range(kc.shape[1]):
            k = torch.cat([pk[j], kc[b, j, :n]]).double()
            v = torch.cat([pv[j], vc[b, j, :n]]).double()
            if not len(k):
                continue
            r = slice(j * G, (j + 1) * G)
            p = torch.softmax(q[b, r].double() @ k.T / math.sqrt(q.shape[2]), 1)
            out[b, r] = p @ v
            tol[b, r] = h * out[b, r].abs() + (h + SLOP) * (p @ v.abs()) + tiny * (1 + len(k) * v.abs().max())
    return out, tol


@pytest.mark.parametrize("B,hq,hkv,d,smax,P,lens", [
    (1, 4, 2, 64, 16, 7, [0]), (3, 32, 8, 128, 300, 100, [0, 300, 33]),      # one workgroup walks both
    (4, 8, 2, 64, 700, 129, [1, 700, 256, 0]), (2, 14, 2, 128, 64, 1000, [64, 3]),  # at most 32 rows a key head
    (40, 8, 4, 128, 300, 515, [0, 300, 257, 256] * 10), (33, 4, 4, 64, 16, 4000, [16, 0, 5] * 11),
    (70, 12, 4, 64, 260, 1030, [260, 1] * 35), (9, 32, 1, 128, 600, 300, [600, 0, 1] * 3),  # row tiles of 128
    (3, 4, 4, 64, 900, 0, [0, 900, 5]), (40, 8, 8, 64, 1000, 9000, [1000, 0, 3, 700] * 10),
    (5, 64, 8, 64, 0, 600, [0] * 5), (2, 4, 4, 128, 0, 9, [0, 0]),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prefix_attention(B, hq, hkv, d, smax, P, lens, dtype):
    g = torch.Generator(device="cuda").manual_seed(B + P)
    q = _rnd(g, B, hq, d, dtype=dtype)
    room = torch.full((2, hkv, P + 5, d), float("nan"), device="cuda", dtype=dtype)  # the prefix inside a longer buffer
    room[:, :, :P] = _rnd(g, 2, hkv, P, d, dtype=dtype)
    kc, vc = _rnd(g, B, hkv, smax, d, dtype=dtype), _rnd(g, B, hkv, smax, d, dtype=dtype)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):  # what lies past a row's length is never looked at
        kc[b, :, n:], vc[b, :, n:] = float("nan"), float("inf")
    att = dec.PrefixDecodeAttention(B, hq, hkv, d, smax, P, "cuda", dtype=dtype)
    got = att(q, room[0, :, :P], room[1, :, :P], kc, vc, ln)
    _within(got, *_exact_prefix(q, room[0, :, :P], room[1, :, :P], kc, vc, ln), "o")
    # other strides, lengths out of range, again: the same bits
    ln2 = torch.where(ln == smax, ln + 77, torch.where(ln == 0, ln - 3, ln)).to(torch.int32)
    again = att(q, room[0, :, :P].contiguous(), room[1, :, :P], kc, vc, ln2)
    assert torch.equal(got, again)


@pytest.mark.parametrize("P", [0, 513])
def test_prefix_attention_of_many_sequences(P):
    """Workgroups that take several chunks each, counted over several groups of 64 sequences, long and empty ones."""
    g = torch.Generator(device="cuda").manual_seed(P)
    B, hq, hkv, d, smax = 331, 8, 4, 64, 530
    lens = [(0, 530, 1, 256, 257, 0, 40)[(b * b + b // 64) % 7] if not 128 <= b < 200 else 0 for b in range(B)]
    q, pk, pv = _rnd(g, B, hq, d), _rnd(g, hkv, P, d), _rnd(g, hkv, P, d)
    kc, vc = _rnd(g, B, hkv, smax, d), _rnd(g, B, hkv, smax, d)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    att = dec.PrefixDecodeAttention(B, hq, hkv, d, smax, P, "cuda")
    for _ in range(2):
        _within(att(q, pk, pv, kc, vc, ln), *_exact_prefix(q, pk, pv, kc, vc, ln), "o")
        ln = ln.flip(0).contiguous()


def test_prefix_attention_growing_scores_and_replays():
    g = torch.Generator(device="cuda").manual_seed(3)
    B, hq, hkv, d, smax, P = 20, 16, 4, 64, 600, 2000
    q = _rnd(g, B, hq, d, scale=3.0)
    grow = torch.linspace(0.1, 5, P, device="cuda")[None, :, None]
    pk, pv = (torch.randn(hkv, P, d, device="cuda", generator=g) * grow).bfloat16(), _rnd(g, hkv, P, d)
    kc, vc = _rnd(g, B, hkv, smax, d), _rnd(g, B, hkv, smax, d)
    lens = torch.full((B,), 600, dtype=torch.int32, device="cuda")
    att = dec.PrefixDecodeAttention(B, hq, hkv, d, smax, P, "cuda")
    _within(att(q, pk, pv, kc, vc, lens), *_exact_prefix(q, pk, pv, kc, vc, lens), "o")
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:  # two graphs of one object
        with torch.cuda.graph(graph):
            outs.append(att(q, pk, pv, kc, vc, lens))
    streams = [torch.cuda.Stream() for _ in graphs]
    for n in (600, 0, 1, 333):
        lens.fill_(n)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):  # replayed at the same time
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        want = att(q, pk, pv, kc, vc, lens)
        assert all(torch.equal(o, want) for o in outs), n


def test_prefix_attention_gpu_refusals():
    for bad in ((1, 4, 2, 32, 8, 8), (1, 66, 2, 64, 8, 8)):
        with pytest.raises(ValueError):
            dec.PrefixDecodeAttention(*bad, "cuda")
    with pytest.raises(ValueError):
        dec.PrefixDecodeAttention(1, 4, 2, 64, 8, 8, "cuda", dtype=torch.float32)
    att = dec.PrefixDecodeAttention(1, 4, 2, 64, 8, 8, "cuda")
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(ValueError):
        att(z(1, 4, 64), z(2, 8, 64), z(2, 8, 64), z(1, 2, 8, 64), z(1, 2, 64, 8).transpose(2, 3),
            torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        att(z(1, 4, 64), z(2, 8, 64), z(2, 8, 64), z(1, 2, 8, 64), z(1, 2, 8, 64), torch.zeros(1, dtype=torch.int32))
