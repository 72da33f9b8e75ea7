"""What the operators on packed and prefix-sharing batches refuse rather than answer wrongly."""
import pytest
import torch
from torch.autograd import forward_ad

from kgwe.ops import attention_packed, norm_rope_qkv
from kgwe.ops import decode as dec
from kgwe.ops import reference as ref
from kgwe.ops.packed import PackedBatch


def _dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


# ------------------------------------------------------------------ forward-mode derivatives
def test_forward_only_calls_refuse_tangents():
    att = dec.PrefixDecodeAttention(1, 4, 2, 16, 8, 5, "cpu", dtype=torch.float32)
    q, p, c = torch.zeros(1, 4, 16), torch.zeros(2, 5, 16), torch.zeros(1, 2, 8, 16)
    lens = torch.zeros(1, dtype=torch.int32)
    hq, hkv, d = 2, 1, 32
    qkv = torch.randn(3, (hq + 2 * hkv) * d)
    cos, sin = ref.rope_tables(8, d)
    pos, w = torch.zeros(3, dtype=torch.int32), torch.ones(d)
    kc, vc = torch.zeros(3, hkv, 8, d), torch.zeros(3, hkv, 8, d)
    with forward_ad.dual_level():
        att(q, p, p, c, c, lens)  # a level alone is nothing to refuse
        for bad in (lambda: att(_dual(q), p, p, c, c, lens), lambda: att(q, p, _dual(p), c, c, lens),
                    lambda: dec.norm_rope_append(_dual(qkv), pos, cos, sin, kc, vc, hq, hkv, d),
                    lambda: dec.norm_rope_append(qkv, pos, cos, sin, kc, vc, hq, hkv, d, _dual(w), w)):
            with pytest.raises(ValueError):
                bad()
            with pytest.raises(ValueError), torch.no_grad():  # which leaves forward mode as it is
                bad()


@pytest.mark.gpu
def test_gpu_kernels_refuse_tangents():
    """A tensor with a tangent does not require a gradient; the kernels would drop the tangent."""
    hq, hkv, d = 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, pk = (torch.randn(s, h, d, device="cuda", generator=g).bfloat16()
                   for s, h in ((5, hq), (5, hkv), (5, hkv), (hkv, 3)))
    qkv, w = torch.randn(5, (hq + 2 * hkv) * d, device="cuda", generator=g).bfloat16(), torch.ones(
        d, device="cuda", dtype=torch.bfloat16)
    batch = PackedBatch([5])
    cos, sin = ref.rope_tables(5, d, device="cuda")
    with forward_ad.dual_level():
        for bad in (lambda: attention_packed(_dual(q), k, v, batch), lambda: attention_packed(q, k, _dual(v), batch),
                    lambda: attention_packed(q, k.clone().requires_grad_(), _dual(v), batch),
                    lambda: attention_packed(q, k, v, batch, prefix=(pk, _dual(pk))),
                    lambda: norm_rope_qkv(_dual(qkv), cos, sin, 5, hq, hkv, d),
                    lambda: norm_rope_qkv(qkv, cos, sin, 5, hq, hkv, d, w, _dual(w)),
                    lambda: norm_rope_qkv(qkv, _dual(cos), sin, 5, hq, hkv, d)):
            with pytest.raises(ValueError):
                bad()
            with pytest.raises(ValueError), torch.no_grad():
                bad()
        attention_packed(q, k, v, batch)


# ------------------------------------------------------------------ a rectangular batch
def test_a_rectangular_batch_fits_its_tables():
    """A sequence length in the place of positions is known on the host: rows past the tables are an undersized table,
    not padding, and the rows are whole sequences (as rope_qkv has it)."""
    hq, hkv, d = 2, 1, 32
    qkv = torch.randn(12, (hq + 2 * hkv) * d)
    cos, sin = ref.rope_tables(8, d)
    for S, offset in ((12, 0), (6, 3), (9, 0), (5, 0), (8, 0)):
        with pytest.raises(ValueError):
            norm_rope_qkv(qkv, cos, sin, S, hq, hkv, d, offset=offset)
    for S, offset in ((6, 2), (4, 0), (1, 7)):
        assert all(t.any(-1).all() for t in norm_rope_qkv(qkv, cos, sin, S, hq, hkv, d, offset=offset))
    assert norm_rope_qkv(qkv[:0], cos, sin, 8, hq, hkv, d)[0].shape == (0, hq, d)


# ------------------------------------------------------------------ caches without room
@pytest.mark.parametrize("T,R,smax", [(3, 3, 0), (3, 0, 8), (0, 0, 8), (0, 3, 0)])
def test_an_empty_cache_is_refused_as_such(T, R, smax):
    hq, hkv, d = 2, 1, 32
    cos, sin = ref.rope_tables(8, d)
    kc, vc = torch.zeros(R, hkv, smax, d), torch.zeros(R, hkv, smax, d)
    ints = torch.zeros(T, dtype=torch.int32)
    with pytest.raises(ValueError, match="no room"):
        dec.norm_rope_append(torch.randn(T, (hq + 2 * hkv) * d), ints, cos, sin, kc, vc, hq, hkv, d, rows=ints)


@pytest.mark.gpu
def test_gpu_append_of_no_rows():
    hq, hkv, d = 2, 1, 64
    cos, sin = ref.rope_tables(8, d, device="cuda")
    kc, vc = torch.ones(2, 3, hkv, 8, d, device="cuda", dtype=torch.bfloat16).unbind()
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    out = dec.norm_rope_append(torch.zeros(0, (hq + 2 * hkv) * d, device="cuda", dtype=torch.bfloat16), none, cos, sin,
                               kc, vc, hq, hkv, d, rows=none, keep_kv=True)
    assert [t.shape for t in out] == [(0, hq, d), (0, hkv, d), (0, hkv, d)] and (kc == 1).all() and (vc == 1).all()


# ------------------------------------------------------------------ plans and captures
@pytest.mark.gpu
def test_host_lengths_are_refused_inside_a_capture():
    """Their copy would break the capture; the refusal leaves it whole."""
    lengths = torch.tensor([3, 2], dtype=torch.int32, device="cuda")
    q = torch.randn(5, 2, 64, device="cuda").bfloat16()
    want = attention_packed(q, q, q, PackedBatch([3, 2]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError):
            PackedBatch([3, 2])
        got = attention_packed(q, q, q, PackedBatch(lengths, total=5))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
