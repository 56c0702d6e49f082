"""The decoder's options on the language-model operators: windowed and rotary
training, padded batches, distillation, prefill and cached decoding, and the
data-parallel harness over them."""
import dataclasses

import pytest
import torch
import torch.nn.functional as F

import lm_reference as ref
from cail_b200.models import GPT2, GPT2Config

E = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def built(build):
    from cail_b200.ops import ext

    ext.build_ops()


def config(**kw):
    return dataclasses.replace(GPT2Config.tiny(), **kw)


def test_default_model_is_unchanged():
    torch.manual_seed(0)
    m = GPT2(GPT2Config.tiny())
    names = [n for n, _ in m.named_parameters()]
    assert names[:3] == ["wte.weight", "wpe.weight", "blocks.0.ln1.weight"] and len(names) == 28
    assert "wpe.weight" not in dict(GPT2(config(rotary=8)).named_parameters())
    idx = torch.randint(0, 512, (2, 64))
    assert m(idx).shape == (2, 64, 512) and m(idx, idx).dim() == 0


def test_refusals_on_cpu():
    m = GPT2(config(window=8, sinks=2))
    with pytest.raises(ValueError, match="CUDA"):
        m(torch.zeros(1, 4, dtype=torch.int64))
    with pytest.raises(ValueError, match="learned positions"):
        m.new_cache(1, 65)
    cache = m.new_cache(2, 4)
    with pytest.raises(ValueError, match="do not fit"):
        m.prefill(torch.zeros(2, 5, dtype=torch.int64), cache)
    with pytest.raises(ValueError, match="one token"):
        m.decode(torch.zeros(3, dtype=torch.int64), cache)
    cache.filled = 4
    with pytest.raises(ValueError, match="full"):
        m.decode(torch.zeros(2, dtype=torch.int64), cache)
    with pytest.raises(ValueError, match="empty"):
        m.prefill(torch.zeros(2, 3, dtype=torch.int64), cache)
    assert GPT2(config(rotary=8)).new_cache(1, 500).length == 500


def test_rotary_plans_belong_to_no_mode():
    """A plan made under inference_mode serves training; a model's plan is there once it is built or moved."""
    from cail_b200 import ops

    m = GPT2(config(rotary=8))
    assert set(m._plans) == {torch.device("cpu")}
    m.to("meta")
    assert set(m._plans) == {torch.device("cpu"), torch.device("meta")}
    with torch.inference_mode():
        plans = [ops.Rotary(8, device="cpu"), ops.Rotary(8, device="cpu").to("meta"), GPT2(config(rotary=8))._plan(torch.device("cpu"))]
    assert not any(p.turns.is_inference() for p in plans)
    assert "_plans" not in GPT2(config()).__dict__


def plain_logits(m, idx, lengths=None):
    """The model in 64 bits, from its parameters, by the operators' plain forms."""
    c, p = m.c, {n: q.detach().double().requires_grad_() for n, q in m.named_parameters()}
    b, t = idx.shape
    x = p["wte.weight"][idx]
    if c.rotary == 0:
        x = x + p["wpe.weight"][:t]
    plan = m._plan(torch.device("cpu")) if c.rotary else None
    f = [float(v) * 2 * torch.pi for v in plan.turns] if plan else None
    at = torch.arange(t, device=idx.device).expand(b, t)
    for i in range(c.n_layer):
        w = lambda n: p[f"blocks.{i}.{n}"]  # noqa: E731
        y = F.layer_norm(x, (c.d_model,), w("ln1.weight"), w("ln1.bias"))
        q, k, v = (z.view(b, t, c.n_head, -1) for z in F.linear(y, w("qkv.weight"), w("qkv.bias")).split(c.d_model, 2))
        if plan:
            q, k = (ref.rotate(z, at, f, plan.amplitude, c.rotary_interleaved) for z in (q, k))
        a = ref.attention(q, k, v, c.window or t, c.sinks, lengths)
        x = x + F.linear(a.reshape(b, t, -1), w("proj.weight"), w("proj.bias"))
        y = F.layer_norm(x, (c.d_model,), w("ln2.weight"), w("ln2.bias"))
        x = x + F.linear(F.gelu(F.linear(y, w("fc.weight"), w("fc.bias")), approximate="tanh"), w("out.weight"), w("out.bias"))
    return F.linear(F.layer_norm(x, (c.d_model,), p["ln_f.weight"], p["ln_f.bias"]), p["wte.weight"]), p


OPTIONS = [dict(window=9, sinks=2), dict(rotary=16), dict(window=20, sinks=0, rotary=8, rotary_interleaved=True),
           dict(window=5, sinks=70, rotary=12, rotary_scaling="parts", rotary_factor=4.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", OPTIONS, ids=str)
def test_training_step_matches_64_bit(kw):
    """Two layers in float32: about 40 roundings lie between the parameters and
    a logit, and as many back, each at most e of values whose norm a
    LayerNorm keeps: 512 e for the logits, 4096 e for the gradients (which sum
    over the tokens with cancellation)."""
    torch.manual_seed(1)
    m = GPT2(config(**kw)).cuda()
    g = torch.Generator().manual_seed(2)
    idx, tgt = (torch.randint(0, 512, (2, 64), generator=g).cuda() for _ in range(2))
    logits = m(idx)
    want, p = plain_logits(m, idx)
    assert ref.rel(logits, want) <= 512 * E
    m(idx, tgt).backward()
    F.cross_entropy(want.flatten(0, 1), tgt.flatten()).backward()
    for n, q in m.named_parameters():
        if n.endswith("qkv.bias"):  # the keys' bias moves no softmax: its gradient is zero but for roundings
            d = m.c.d_model
            q.grad[d:2 * d] = 0
            p[n].grad[d:2 * d] = 0
        assert ref.rel(q.grad, p[n].grad) <= 4096 * E, n


@pytest.mark.gpu
def test_padded_batch_and_distillation_match_64_bit():
    torch.manual_seed(3)
    m = GPT2(config(window=11, sinks=3, rotary=16)).cuda()
    g = torch.Generator().manual_seed(4)
    idx, tgt = (torch.randint(0, 512, (3, 50), generator=g).cuda() for _ in range(2))
    lengths = torch.tensor([50, 31, 1], dtype=torch.int32).cuda()
    for b, n in enumerate(lengths.tolist()):
        tgt[b, n:] = -100
    ids = torch.randint(0, 512, (3, 50, 6), generator=g).cuda()
    top = torch.randn(3, 50, 6, generator=g).cuda()
    loss = m(idx, tgt, teacher=(ids, top), temperature=2.0, hard_weight=0.3, lengths=lengths)
    loss.backward()
    want, p = plain_logits(m, idx, lengths)
    wloss = ref.distill(want.flatten(0, 1), ids.flatten(0, 1), top.flatten(0, 1), tgt.flatten(), 2.0, 0.3)
    wloss.backward()
    assert abs(float(loss.detach()) - float(wloss.detach())) <= 512 * E * float(wloss.detach())
    for n, q in m.named_parameters():
        if not n.endswith("qkv.bias"):
            assert ref.rel(q.grad, p[n].grad) <= 4096 * E, n


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[50, 31, 1], [0, 7, 50], None], ids=str)
def test_distillation_without_targets_leaves_padding_out(lengths):
    """The teacher alone over a padded batch: the mean is over the sequences' tokens, whatever lies behind them."""
    torch.manual_seed(3)
    m = GPT2(config(window=11, sinks=3, rotary=16)).cuda()
    g = torch.Generator().manual_seed(5)
    idx = torch.randint(0, 512, (3, 50), generator=g).cuda()
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32).cuda()
    ids = torch.randint(0, 512, (3, 50, 6), generator=g).cuda()
    top = torch.randn(3, 50, 6, generator=g).cuda()
    got = m(idx, teacher=(ids, top), temperature=2.0, hard_weight=0.7, lengths=n)
    got.backward()
    want, p = plain_logits(m, idx, n)
    rows = torch.cat([torch.arange(50) + 50 * b for b in range(3)] if n is None else [torch.arange(k) + 50 * b for b, k in enumerate(lengths)]).cuda()
    wloss = ref.distill(want.flatten(0, 1)[rows], ids.flatten(0, 1)[rows], top.flatten(0, 1)[rows], None, 2.0, 0.0)
    wloss.backward()
    assert abs(float(got.detach()) - float(wloss.detach())) <= 512 * E * float(wloss.detach())
    for name, q in m.named_parameters():
        if not name.endswith("qkv.bias"):
            assert ref.rel(q.grad, p[name].grad) <= 4096 * E, name
    if n is not None:  # what the padding holds is nothing to the loss
        for b, k in enumerate(lengths):
            idx[b, k:], ids[b, k:], top[b, k:] = 3, 5, float("nan")
        assert torch.equal(m(idx, teacher=(ids, top), temperature=2.0, lengths=n), got)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict()] + OPTIONS, ids=str)
def test_prefill_and_decode_follow_forward(kw):
    """Prompts of unequal length, then tokens one by one: the logits of the
    whole sequences in one pass (the same sums in another order: 1024 e)."""
    torch.manual_seed(5)
    m = GPT2(config(**kw)).cuda()
    g = torch.Generator().manual_seed(6)
    idx = torch.randint(0, 512, (3, 60), generator=g).cuda()
    lengths = torch.tensor([40, 17, 1], dtype=torch.int32).cuda()
    cache = m.new_cache(3)
    with torch.no_grad():
        want = [m(idx[b:b + 1])[0] for b in range(3)]
    got = m.prefill(idx[:, :40], cache, lengths)
    rows = torch.arange(3).cuda()
    for step in range(21):
        for b in range(3):
            assert ref.rel(got[b], want[b][int(lengths[b]) + step - 1]) <= 1024 * E, (step, b)
        if step < 20:
            got = m.decode(idx[rows, cache.lengths.long()], cache)
    with pytest.raises(ValueError, match="full"):
        for _ in range(10):
            m.decode(idx[:, 0], cache)


@pytest.mark.gpu
def test_decode_under_autocast():
    """bf16 keys and values into a float32 cache: forward's logits, to bf16's roundings (10 of 2^-8 deep)."""
    torch.manual_seed(8)
    m = GPT2(config(rotary=16, window=50, sinks=2)).cuda()
    idx = torch.randint(0, 512, (2, 40)).cuda()
    cache = m.new_cache(2)
    with torch.autocast("cuda", torch.bfloat16):
        out = m.prefill(idx[:, :35], cache)
        for t in range(35, 40):
            out = m.decode(idx[:, t], cache)
    with torch.no_grad():
        assert ref.rel(out, m(idx)[:, 39]) <= 10 * 2.0 ** -8


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [0, 16])
def test_captured_decode(rotary):
    """Replays append tokens as eager calls do; past the cache's length they stay inside it."""
    torch.manual_seed(9)
    m = GPT2(config(rotary=rotary, window=20, sinks=2)).cuda()
    idx = torch.randint(0, 512, (2, 30)).cuda()
    eager, cache = m.new_cache(2, 30), m.new_cache(2, 30)
    m.prefill(idx[:, :10], eager)
    m.prefill(idx[:, :10], cache)
    static = idx[:, 10].clone()
    m.decode(static, m.new_cache(2, 30))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.decode(static, cache)
    for t in range(10, 30):
        static.copy_(idx[:, t])
        graph.replay()
        want = m.decode(idx[:, t], eager)
        assert torch.equal(out, want)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a[:, :29], b[:, :29]) for a, b in zip(cache.k, eager.k))


@pytest.mark.gpu
def test_training_after_inference_mode():
    """The same gradients whether or not the model's first call was under inference_mode, and a first call under capture."""
    torch.manual_seed(10)
    m = GPT2(config(rotary=16, window=9)).cuda()
    idx = torch.randint(0, 512, (2, 50)).cuda()
    m(idx, idx).backward()
    want = [p.grad.clone() for p in m.parameters()]
    again = GPT2(m.c).cuda()
    again.load_state_dict(m.state_dict())
    with torch.inference_mode():
        again(idx)
        cache = again.new_cache(2)
        again.decode(again.prefill(idx, cache).argmax(-1), cache)
    again(idx, idx).backward()
    for p, w in zip(again.parameters(), want):
        assert ref.rel(p.grad, w) <= 64 * E  # torch's own sums may come in another order
    from cail_b200 import ops

    fresh = GPT2(m.c).cuda()
    q = torch.randn(1, 7, 2, 16, device="cuda")
    ops.rotary(q, None, m._plan(q.device))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rotary(q, None, fresh._plan(q.device))
    graph.replay()
    assert torch.equal(out, ops.rotary(q, None, m._plan(q.device)))


def test_caches_belong_to_no_mode_on_cpu():
    with torch.inference_mode():
        cache = GPT2(config(window=8)).new_cache(2, 4)
    assert not any(t.is_inference() for t in (*cache.k, *cache.v, cache.lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("made, filled, read", [(True, True, False), (True, False, True), (False, True, False)])
def test_caches_belong_to_no_mode(made, filled, read):
    """A cache made, filled and read inside inference_mode or outside, in any mixture: the same logits."""
    torch.manual_seed(11)
    m = GPT2(config(rotary=16, window=9)).cuda()
    idx = torch.randint(0, 512, (2, 20)).cuda()

    def run(made, filled, read):
        with torch.inference_mode(made):
            cache = m.new_cache(2)
        with torch.inference_mode(filled):
            m.prefill(idx[:, :18], cache)
            m.decode(idx[:, 18], cache)
        with torch.inference_mode(read):
            return m.decode(idx[:, 19], cache)

    assert torch.equal(run(made, filled, read), run(False, False, False))


@pytest.mark.gpu
def test_bf16_model_runs_on_the_tensor_cores():
    """A bf16 model of heads of 64: step and decoding run, gradients are finite
    and near the float32 model's (10 roundings of 2^-8 deep)."""
    torch.manual_seed(7)
    c = config(d_model=128, n_head=2, n_ctx=256, window=100, sinks=4, rotary=64)
    m32 = GPT2(c).cuda()
    m = GPT2(c).cuda().bfloat16()
    m32.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    idx = torch.randint(0, 512, (2, 256)).cuda()
    m(idx, idx).backward()
    m32(idx, idx).backward()
    for (n, q), w in zip(m.named_parameters(), m32.parameters()):
        if not n.endswith("qkv.bias"):
            assert ref.rel(q.grad, w.grad) <= 10 * 2.0 ** -8, n
    cache = m.new_cache(2)
    out = m.prefill(idx[:, :200], cache)
    for t in range(200, 205):
        out = m.decode(idx[:, t], cache)
    with torch.no_grad():
        assert ref.rel(out, m(idx)[:, 204]) <= 10 * 2.0 ** -8


@pytest.mark.gpu
def test_data_parallel_harness_over_the_options():
    """Gradients land in the harness' buckets, equal to the same step without it."""
    from cail_b200.parallel import BucketedAllreduce

    torch.manual_seed(8)
    c = config(window=9, sinks=2, rotary=16)
    m, w = GPT2(c).cuda(), GPT2(c).cuda()
    w.load_state_dict(m.state_dict())
    ddp = BucketedAllreduce(m, 1, bucket_bytes=64 << 10)
    g = torch.Generator().manual_seed(9)
    idx, tgt = (torch.randint(0, 512, (2, 64), generator=g).cuda() for _ in range(2))
    ids, top = torch.randint(0, 512, (2, 64, 4), generator=g).cuda(), torch.randn(2, 64, 4, generator=g).cuda()
    for _ in range(2):
        ddp.zero_grad()
        w.zero_grad()
        m(idx, tgt, teacher=(ids, top)).backward()
        ddp.finish()
        ddp.check_views(m)
        w(idx, tgt, teacher=(ids, top)).backward()
        assert all(torch.equal(a.grad, b.grad) or ref.rel(a.grad, b.grad) <= 64 * E for a, b in zip(m.parameters(), w.parameters()))
    ddp.close()
