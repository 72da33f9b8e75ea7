"""Packed batches, attention over them and the q / k norm with rotation:
tables, refusals and CPU references (the GPU kernels: test_packed_gpu.py)."""
import pytest
import torch

from kgwe.ops import attention, attention_packed, norm_rope_qkv, rope_qkv
from kgwe.ops import decode as dec
from kgwe.ops import reference as ref
from kgwe.ops.packed import PackedBatch


def _qkv(T, hq=4, hkv=2, d=64, dtype=torch.float32):
    g = torch.Generator().manual_seed(0)
    return tuple(torch.randn(T, h, d, generator=g).to(dtype) for h in (hq, hkv, hkv))


@pytest.mark.parametrize("lengths,total", [([3, 0, 5], 10), ([], 2), ([0], 0), ([1], 1), ([0, 0, 4, 0], 4)])
def test_batch_tables(lengths, total):
    b = PackedBatch(lengths, total=total, device="cpu")
    starts = [sum(lengths[:i]) for i in range(len(lengths) + 1)]
    assert b.cu.tolist() == starts + [total]
    want_pos = [p for n in lengths for p in range(n)] + [-1] * (total - sum(lengths))
    want_seq = [i for i, n in enumerate(lengths) for _ in range(n)] + [-1] * (total - sum(lengths))
    assert b.positions.tolist() == want_pos and b.seq_ids.tolist() == want_seq
    assert b.last_rows.tolist() == [s - 1 for s in starts[1:]]


@pytest.mark.parametrize("lengths,total", [([-1], None), ([4, 5], 8), ([1], -1), (torch.zeros(2, 2, dtype=torch.int32), 4),
                                           (torch.zeros(2), 4)])
def test_batch_refusals(lengths, total):
    with pytest.raises(ValueError):
        PackedBatch(lengths, total=total, device="cpu")


def test_packed_reference_is_attention_of_each_sequence():
    lengths = [5, 0, 17, 1]
    q, k, v = _qkv(sum(lengths) + 3)
    o = attention_packed(q, k, v, PackedBatch(lengths, total=q.shape[0], device="cpu"))
    at = 0
    for n in lengths:
        if n:
            want = attention(q[None, at:at + n], k[None, at:at + n], v[None, at:at + n])[0]
            assert torch.allclose(o[at:at + n], want, atol=1e-5)
        at += n
    assert not o[at:].any()


def test_packed_reference_with_prefix_is_attention_behind_it():
    q, k, v = _qkv(12 + 7)
    P = 12
    own = attention_packed(q[P:], k[P:], v[P:], PackedBatch([7], device="cpu"),
                           prefix=(k[:P].transpose(0, 1), v[:P].transpose(0, 1)))
    assert torch.allclose(own, attention(q[None], k[None], v[None])[0, P:], atol=1e-5)


def test_attention_packed_refusals():
    q, k, v = _qkv(8)
    b = PackedBatch([8], device="cpu")
    pre = torch.randn(2, 4, 64)
    for bad in (lambda: attention_packed(q[:7], k[:7], v[:7], b), lambda: attention_packed(q, k, v[:, :1], b),
                lambda: attention_packed(q[:, :3], k, v, b), lambda: attention_packed(q, k, v.double(), b),
                lambda: attention_packed(q[..., :32], k, v, b), lambda: attention_packed(q[0], k, v, b),
                lambda: attention_packed(q, k, v, b, prefix=(pre, pre[:, :3])),
                lambda: attention_packed(q, k, v, b, prefix=(pre[:1], pre[:1])),
                lambda: attention_packed(q, k, v, b, prefix=(pre.double(), pre.double())),
                lambda: attention_packed(q.clone().requires_grad_(), k, v, b, prefix=(pre, pre))):
        with pytest.raises(ValueError):
            bad()


def test_rotation_alone_is_rope_qkv():
    S, hq, hkv, d = 6, 4, 2, 32
    qkv = torch.randn(2 * S, (hq + 2 * hkv) * d)
    cos, sin = ref.rope_tables(S, d)
    got = norm_rope_qkv(qkv, cos, sin, PackedBatch([S, S], device="cpu").positions, hq, hkv, d)
    for other in (rope_qkv(qkv, cos, sin, S, hq, hkv, d), norm_rope_qkv(qkv, cos, sin, S, hq, hkv, d)):
        for a, b in zip(got, other):
            assert torch.equal(a, b)


def test_norm_rope_reference_padding_and_offset():
    hq, hkv, d = 2, 1, 32
    qkv = torch.randn(4, (hq + 2 * hkv) * d)
    qkv[3] = float("nan")
    cos, sin = ref.rope_tables(8, d)
    w = torch.ones(d)
    pos = torch.tensor([0, 3, 6, -1], dtype=torch.int32)
    q, k, v = norm_rope_qkv(qkv, cos, sin, pos, hq, hkv, d, w, w, offset=2)
    assert not q[2:].any() and not k[2:].any() and not v[2:].any()  # 6 + 2 is behind the table, -1 padding
    q0, _, _ = norm_rope_qkv(qkv[:2], cos, sin, pos[:2] + 2, hq, hkv, d, w, w)
    assert torch.equal(q[:2], q0)
    assert torch.allclose(q[:2].pow(2).mean(-1), torch.ones(2, hq), atol=1e-3)  # a rotation keeps the norm


def test_append_writes_only_its_places():
    hq, hkv, d, smax = 2, 1, 32, 5
    qkv = torch.randn(4, (hq + 2 * hkv) * d)
    cos, sin = ref.rope_tables(smax, d)
    kc, vc = torch.zeros(3, hkv, smax, d), torch.zeros(3, hkv, smax, d)
    pos = torch.tensor([4, 5, -1, 0], dtype=torch.int32)
    rows = torch.tensor([2, 0, 1, 7], dtype=torch.int32)
    q, k, v = dec.norm_rope_append(qkv, pos, cos, sin, kc, vc, hq, hkv, d, rows=rows, keep_kv=True)
    assert torch.equal(kc[2, :, 4], k[0]) and torch.equal(vc[2, :, 4], v[0])
    kc[2, :, 4] = vc[2, :, 4] = 0
    assert not kc.any() and not vc.any()


def test_norm_rope_refusals():
    hq, hkv, d = 2, 1, 32
    qkv = torch.randn(3, (hq + 2 * hkv) * d)
    cos, sin = ref.rope_tables(8, d)
    pos = torch.zeros(3, dtype=torch.int32)
    w = torch.ones(d)
    kc = torch.zeros(3, hkv, 8, d)
    for bad in (lambda: norm_rope_qkv(qkv[:, 1:], cos, sin, pos, hq, hkv, d),
                lambda: norm_rope_qkv(qkv, cos, sin, pos.long(), hq, hkv, d),
                lambda: norm_rope_qkv(qkv, cos, sin, pos[:2], hq, hkv, d),
                lambda: norm_rope_qkv(qkv, cos, sin, 0, hq, hkv, d),
                lambda: dec.norm_rope_append(qkv.clone().requires_grad_(), pos, cos, sin, kc, kc.clone(), hq, hkv, d),
                lambda: dec.norm_rope_append(qkv, 3, cos, sin, kc, kc.clone(), hq, hkv, d),
                lambda: norm_rope_qkv(qkv, cos, sin, pos, hq, hkv, d, q_weight=w),
                lambda: norm_rope_qkv(qkv, cos, sin, pos, hq, hkv, d, w[:4], w[:4]),
                lambda: norm_rope_qkv(qkv, cos, sin, pos, hq, hkv, d, w.double(), w.double()),
                lambda: norm_rope_qkv(qkv, cos.double(), sin, pos, hq, hkv, d),
                lambda: norm_rope_qkv(qkv, cos[:, :4], sin[:, :4], pos, hq, hkv, d),
                lambda: norm_rope_qkv(qkv, cos, sin, pos, hq, hkv, d, offset=-1),
                lambda: dec.norm_rope_append(qkv, pos, cos, sin, kc, kc, hq, hkv, d),
                lambda: dec.norm_rope_append(qkv, pos, cos[:4], sin[:4], kc, kc.clone(), hq, hkv, d),
                lambda: dec.norm_rope_append(qkv, pos, cos, sin, kc[:2], kc[:2].clone(), hq, hkv, d),
                lambda: dec.norm_rope_append(qkv, pos, cos, sin, kc, kc.clone().double(), hq, hkv, d),
                lambda: dec.norm_rope_append(qkv, pos, cos, sin, kc, kc.clone(), hq, hkv, d, offset=1)):
        with pytest.raises(ValueError):
            bad()


def test_norm_rope_reference_gradient_matches_differences():
    hq, hkv, d = 2, 1, 32
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(3, (hq + 2 * hkv) * d, generator=g).requires_grad_(True)
    cos, sin = ref.rope_tables(8, d)
    pos = torch.tensor([1, 5, -1], dtype=torch.int32)
    w = (1 + 0.2 * torch.randn(2, d, generator=g)).requires_grad_(True)
    dy = [torch.randn(3, h, d, generator=g) for h in (hq, hkv, hkv)]

    def value(x, ww):
        return sum((a * b).sum() for a, b in zip(norm_rope_qkv(x, cos, sin, pos, hq, hkv, d, ww[0], ww[1]), dy))

    value(qkv, w).backward()
    step = torch.randn(qkv.shape, generator=g), torch.randn(w.shape, generator=g)
    h = 1e-2
    with torch.no_grad():
        diff = (value(qkv + h * step[0], w + h * step[1]) - value(qkv - h * step[0], w - h * step[1])) / (2 * h)
    want = (qkv.grad * step[0]).sum() + (w.grad * step[1]).sum()
    assert abs(diff - want) < 2e-2 * max(1.0, abs(want))
    assert not qkv.grad[2].any()


def test_prefix_attention_reference_is_decode_attention_behind_a_prefix():
    B, hq, hkv, d, smax, P = 3, 4, 2, 16, 9, 5
    g = torch.Generator().manual_seed(2)
    q, pk, pv = (torch.randn(*s, generator=g) for s in ((B, hq, d), (hkv, P, d), (hkv, P, d)))
    kc, vc = torch.randn(B, hkv, smax, d, generator=g), torch.randn(B, hkv, smax, d, generator=g)
    lens = torch.tensor([0, 4, 9], dtype=torch.int32)
    got = dec.PrefixDecodeAttention(B, hq, hkv, d, smax, P, "cpu", dtype=torch.float32)(q, pk, pv, kc, vc, lens)
    whole = [torch.cat([p.expand(B, -1, -1, -1), c], 2) for p, c in ((pk, kc), (pv, vc))]
    assert torch.allclose(got, dec.decode_attention_reference(q, *whole, lens + P), atol=1e-5)
    none = dec.PrefixDecodeAttention(B, hq, hkv, d, smax, 0, "cpu", dtype=torch.float32)(
        q, pk[:, :0], pv[:, :0], kc, vc, lens)
    assert not none[0].any()  # a row without any key


def test_prefix_attention_refusals():
    for bad in ((0, 4, 2, 64, 8, 8), (1, 3, 2, 64, 8, 8), (1, 4, 2, 64, 0, 0), (1, 4, 2, 64, -1, 8)):
        with pytest.raises(ValueError):
            dec.PrefixDecodeAttention(*bad, "cpu")
    att = dec.PrefixDecodeAttention(1, 4, 2, 16, 8, 5, "cpu", dtype=torch.float32)
    q, p, c = torch.zeros(1, 4, 16), torch.zeros(2, 5, 16), torch.zeros(1, 2, 8, 16)
    lens = torch.zeros(1, dtype=torch.int32)
    for args in ((q[:, :2], p, p, c, c, lens), (q, p[:, :4], p[:, :4], c, c, lens), (q, p, p, c[:, :, :7], c[:, :, :7], lens),
                 (q, p, p, c, c, lens.long()), (q, p.double(), p, c, c, lens), (q, p, p, c, c, lens[:0]),
                 (q.clone().requires_grad_(), p, p, c, c, lens)):
        with pytest.raises(ValueError):
            att(*args)


def test_rows_that_the_kernels_read_in_place():
    """What is passed on with its strides: dense rows from 16 bytes on, which do not overlap and lie no further apart
    than the kernels' offsets reach; everything else is copied, and a copy has the strides of its shape."""
    from kgwe.ops._lib import rows16, token_view

    x = torch.randn(6, 4, 64, dtype=torch.bfloat16)
    wide = torch.randn(6, 3 * 4 * 64, dtype=torch.bfloat16)
    odd = torch.randn(6, 4 * 64 + 3, dtype=torch.bfloat16)
    for t in (x, x.transpose(0, 1), x[:, :1].expand(6, 4, 64), wide[:, 256:512].view(6, 4, 64)):
        got, at, row, head = token_view(t)
        assert got is t and at == t.data_ptr() and (row, head) == t.stride()[:2]
    overlapping = torch.randn(512, dtype=torch.bfloat16).as_strided((6, 4, 64), (8, 64, 1))
    far = torch.randn((1 << 22) + 200, dtype=torch.bfloat16).as_strided((2, 2, 64), ((1 << 22) + 8, 64, 1))
    for t in (x[:1].expand(6, 4, 64), overlapping, odd[:, :256].view(6, 4, 64), odd[:1, :256].view(1, 4, 64),
              odd[:1, 3:259].view(1, 4, 64), far):
        got, at, row, head = token_view(t)
        assert torch.equal(got, t) and at == got.data_ptr() and at % 16 == 0
        assert (row, head) == tuple(got.stride()[:2]) == (t.shape[1] * 64, 64)
    for t in (x, x.transpose(0, 1), x[:1].expand(6, 4, 64), wide[:, :512], wide[:, :512][:1]):
        assert rows16(t) is t
    for t in (odd[:1, :256], odd[:, 8:264], wide[:1, :256].expand(6, 256), x[:, :1].expand(6, 4, 64),
              x[0, :1].expand(4, 64)[None], overlapping.transpose(0, 1), far.transpose(0, 1)):
        got = rows16(t)
        assert torch.equal(got, t) and got.data_ptr() % 16 == 0 and got.is_contiguous()
        assert got.stride() == torch.empty(t.shape).stride()
