"""Packed batches and shared prefixes through the model, the generator, the
batch server and the trainer: each has to be the same computation as the
sequences one by one."""
import dataclasses
import threading
import time

import pytest
import torch

from kgwe.models import llama
from kgwe.models.infer import Generator
from kgwe.ops.packed import PackedBatch
from kgwe.serving import client
from kgwe.serving.batch_server import BatchServer

TINY = llama.PRESETS["tiny"]
QKN = dataclasses.replace(TINY, name="tiny-qk-norm", qk_norm=True)


def _model(cfg, device="cpu", dtype=torch.float32):
    torch.manual_seed(5)
    m = llama.build(cfg, device=device, dtype=dtype)
    if cfg.qk_norm:
        with torch.no_grad():
            for layer in m.layers:
                for w in (layer.attention.q_norm, layer.attention.k_norm):
                    w.copy_((1 + 0.2 * torch.randn(w.shape)).to(w))
    return m


@pytest.fixture(scope="module", params=[TINY, QKN], ids=["plain", "qk_norm"])
def model(request):
    return _model(request.param).eval()


def _prompts(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, TINY.vocab_size, (n,), generator=g) for n in lens]


def test_packed_logits_and_gradients_are_those_of_each_document(model):
    docs = _prompts([9, 1, 20, 6])
    pad = torch.zeros(3, dtype=torch.long)
    tokens = torch.cat([*docs, pad])
    batch = PackedBatch([len(d) for d in docs], total=len(tokens), device="cpu")
    labels = torch.full_like(tokens, -100)
    at, total, count = 0, 0.0, 0
    model.zero_grad()
    for d in docs:
        if len(d) > 1:
            labels[at:at + len(d) - 1] = d[1:]
            loss = model(d[None, :-1], d[None, 1:]) * (len(d) - 1)
            loss.backward()
            total, count = total + loss.item(), count + len(d) - 1
        at += len(d)
    want = {n: p.grad / count for n, p in model.named_parameters()}
    model.zero_grad()
    loss = model(tokens, labels, batch)
    loss.backward()
    assert abs(loss.item() - total / count) < 1e-4
    for n, p in model.named_parameters():
        assert torch.allclose(p.grad, want[n], atol=1e-5 + 1e-3 * want[n].abs().max().item()), n
    model.zero_grad()
    logits = model(tokens, batch=batch)[0]
    at = 0
    for d in docs:
        assert torch.allclose(logits[at:at + len(d)], model(d[None])[0], atol=1e-4)
        at += len(d)


def test_packed_batch_must_fit_the_tokens(model):
    with pytest.raises(ValueError):
        model(torch.zeros(7, dtype=torch.long), batch=PackedBatch([4], device="cpu"))


def test_generator_decodes_like_the_full_forward(model):
    """Prefill + steps with q / k norms, against the whole sequence through the model."""
    prompt = torch.stack(_prompts([11, 11]))
    gen = Generator(model, 2, 24)
    out = gen.generate(prompt, 6)
    seq = prompt
    for i in range(6):
        nxt = model(seq)[:, -1].argmax(-1)
        assert torch.equal(out[:, i], nxt)
        seq = torch.cat([seq, nxt[:, None]], 1)


def test_packed_prefill_is_prefill_of_each_prompt(model):
    lens = [5, 17, 1, 9]
    prompts = _prompts(lens)
    gen = Generator(model, 5, 32)
    gen.idle_rows(1, 2)
    rows = [3, 0, 4, 2]
    first = gen.prefill_packed(prompts, rows)
    steps = [gen.step().clone() for _ in range(5)]
    for i, r in enumerate(rows):
        one = Generator(model, 1, 32)
        want = one.generate(prompts[i][None], 6)[0].tolist()
        assert [int(first[i])] + [int(s[r]) for s in steps] == want
    for bad in (([prompts[0]], [0, 1]), ([prompts[0]] * 2, [1, 1]), ([prompts[0]], [5]), ([prompts[0][:0]], [0]),
                ([torch.zeros(32, dtype=torch.long)], [0]), ([], [])):
        with pytest.raises(ValueError):
            gen.prefill_packed(*bad)


def test_prefix_generator_is_the_generator_of_whole_prompts(model):
    prefix, prompts = _prompts([13], seed=3)[0], _prompts([4, 7], seed=4)
    gen = Generator(model, 2, 20, prefix=prefix.tolist())
    first = gen.prefill_packed(prompts, [0, 1])
    steps = [gen.step().clone() for _ in range(4)]
    rect = Generator(model, 2, 20, prefix=prefix)  # the rectangular call goes the same way
    both = rect.generate(torch.stack([prompts[0], prompts[1][:4]]), 5)
    for r in range(2):
        want = Generator(model, 1, 40).generate(torch.cat([prefix, prompts[r]])[None], 5)[0].tolist()
        assert [int(first[r])] + [int(s[r]) for s in steps] == want
    assert both[0].tolist() == Generator(model, 1, 40).generate(torch.cat([prefix, prompts[0]])[None], 5)[0].tolist()
    with pytest.raises(ValueError):
        Generator(model, 1, 8, prefix=torch.zeros(2, 2, dtype=torch.long))


@pytest.mark.parametrize("prefix", [None, [7, 8, 9, 10, 11]])
def test_server_admits_requests_of_all_lengths_in_one_pass(prefix):
    m = _model(TINY).eval()
    srv = BatchServer(m, 4, 2, 96, flush=4, graph=False, packed=True, prefix=prefix)
    addr = srv.listen("127.0.0.1:0")  # accepting, not serving yet: the requests queue up
    reqs = [([p.tolist() for p in _prompts(lens, seed=sum(lens))], n)
            for lens, n in (((16, 16), 7), ((3, 30), 5), ((24, 1), 3))]
    out = [None] * len(reqs)
    ths = [threading.Thread(target=lambda i=i: out.__setitem__(i, client.generate(reqs[i][0], reqs[i][1], addr)))
           for i in range(len(reqs))]
    [x.start() for x in ths]
    deadline = time.time() + 10
    while srv.pending.qsize() < len(reqs) and time.time() < deadline:
        time.sleep(0.01)
    t = threading.Thread(target=srv.serve_forever, daemon=True)
    t.start()
    try:
        [x.join(60) for x in ths]
        for (prompt, n), res in zip(reqs, out):
            for row, got in zip(prompt, res["tokens"]):
                whole = torch.tensor((prefix or []) + row)[None]
                assert got == Generator(m, 1, 128).generate(whole, n)[0].tolist()
        st = client.call(addr, {"op": "stats"})
        assert st["served"] == 3 and st["prefill_passes"] == 1 and st["prefix_tokens"] == len(prefix or [])
        bad = client.call(addr, {"op": "generate", "prompt": [[1], [2] * 95], "new": 2})
        assert "error" in bad
    finally:
        srv.stop()
        t.join(5)
    with pytest.raises(ValueError):
        BatchServer(m, 1, 1, 16, graph=False, prefix=[TINY.vocab_size])


def test_trainer_on_packed_documents():
    from kgwe.bench.train import TrainConfig, Trainer
    from kgwe.parallel import dist as kdist

    info = kdist.init()
    cfg = TrainConfig(model="tiny", seq_len=64, micro_batch=2, parallel="zero", doc_len=40)
    tr = Trainer(cfg, info)
    lens = tr.doc_lengths()
    assert sum(lens) == 128 and max(lens) <= 40 and lens == Trainer(cfg, info).doc_lengths()
    before = [p.detach().clone() for p in tr.model.parameters()]
    loss = tr.step()
    assert torch.isfinite(loss) and any(not torch.equal(a, b) for a, b in zip(before, tr.model.parameters()))
    assert lens != tr.doc_lengths()
    with pytest.raises(ValueError):
        Trainer(dataclasses.replace(cfg, doc_len=1), info)


# ------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("cfg", [TINY, QKN], ids=["plain", "qk_norm"])
def test_gpu_packed_training_step_against_the_cpu(cfg):
    """Gradients in bf16 on the GPU next to fp32 on the CPU, weight by weight.
    About 24 roundings to bf16 lie between the embedding and the loss and as
    many on the way back, each at most 2^-8 relative and of random sign:
    sqrt(48) 2^-8 / sqrt(3) = 1.6e-2 expected, three times that allowed."""
    m, c = _model(cfg, "cuda", torch.bfloat16), _model(cfg)
    c.load_state_dict({k: v.float().cpu() for k, v in m.state_dict().items()})
    lens = [70, 1, 130, 33]
    tokens = torch.cat([*_prompts(lens), torch.zeros(6, dtype=torch.long)])
    labels = torch.cat([tokens[1:], tokens[:1]])
    batch = PackedBatch(lens, total=len(tokens), device="cpu")
    labels[batch.last_rows.long()] = -100
    labels[sum(lens):] = -100
    want = c(tokens, labels, batch)
    want.backward()
    got = m(tokens.cuda(), labels.cuda(), PackedBatch(lens, total=len(tokens)))
    got.backward()
    assert abs(got.item() - want.item()) < 2e-2
    for (n, a), (_, b) in zip(m.named_parameters(), c.named_parameters()):
        rel = ((a.grad.float().cpu() - b.grad).norm() / b.grad.norm()).item()
        assert rel < 5e-2, (n, rel)


@pytest.mark.gpu
@pytest.mark.parametrize("cfg", [TINY, QKN], ids=["plain", "qk_norm"])
@pytest.mark.parametrize("prefix_len", [0, 37])
@pytest.mark.parametrize("batch", [3, 12])
def test_gpu_generator_logits_match_full_forward(cfg, prefix_len, batch):
    """Packed prefill and graph-replayed steps behind a prefix: logits of every
    step next to the whole sequences in fp32 on the CPU, over the tokens that the GPU chose.
    About 24 roundings to bf16 to the logits, each at most 2^-8 relative and of random sign:
    sqrt(24) 2^-8 / sqrt(3) = 1.1e-2 expected, three times that allowed."""
    m, c = _model(cfg, "cuda", torch.bfloat16).eval(), _model(cfg).eval()
    c.load_state_dict({k: v.float().cpu() for k, v in m.state_dict().items()})
    prefix = _prompts([prefix_len], seed=1)[0]
    prompts = _prompts([(7 * i) % 23 + 1 for i in range(batch)], seed=2)
    gen = Generator(m, batch, 64, keep_logits=True, prefix=prefix if prefix_len else None)
    tok = gen.prefill_packed(prompts, list(range(batch))).cpu()
    seqs = [torch.cat([prefix, p]) for p in prompts]
    logits = gen.logits.float().cpu()
    gen.logits = None
    for step in range(4):
        with torch.no_grad():
            want = torch.stack([c(s[None])[0, -1] for s in seqs])
        rel = ((logits - want).norm() / want.norm()).item()
        assert rel < 3e-2, (step, rel)
        seqs = [torch.cat([s, t[None]]) for s, t in zip(seqs, tok)]
        if step == 0:
            gen.capture()
        tok = gen.step().cpu().clone()
        logits = gen.logits.float().cpu()
