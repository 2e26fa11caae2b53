"""The serving and distillation operators as the policy uses them: 8-bit decode caches, drafted decoding, a student's training step."""
import pytest
import torch

from serving_ref import distill

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _policy(seed=0, d=64, layers=2, heads=2, ctx=96, **kw):
    from neko_amd.policy.gato_policy import GatoPolicy
    torch.manual_seed(seed)
    m = GatoPolicy(DEV, d, layers, heads, 0.0, resid_mid_channels=128, context_len=ctx, text_tokenizer=128, **kw)
    m.transformer.drop.p = 0.0
    m.eval()
    with torch.no_grad():      # attention that matters and logits that differ: random initial weights leave both near zero
        for n, p in m.named_parameters():
            if "c_attn.weight" in n or "c_proj.weight" in n or "predict_token" in n or "embed_token" in n:
                p.mul_(6.0)
    m._flat.ensure_shadow()
    return m


def _prompt(n, seed=1):
    return {"text": torch.randint(0, 128, (n,), generator=torch.Generator().manual_seed(seed)).tolist()}


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("d,heads", [(64, 2), (128, 2), (256, 2)])
def test_decoder_attends_to_what_the_cache_holds(kind, d, heads):
    """One attention step of KV8Decoder against a 64-bit attention over the bf16 rows that kv8_read returns; extension by many rows and by few."""
    from neko_amd import engine, ops
    from serving_ref import attention
    m = _policy(d=d, heads=heads)
    m.kv_cache = kind
    dec = m._new_decoder(96, torch.device(DEV))
    assert isinstance(dec, engine.KV8Decoder)
    g = torch.Generator().manual_seed(d)
    H, hd, n = heads, d // heads, 0
    for T in (40, 5, 1, 8, 1):
        rows = torch.randn(T, 3 * d, generator=g).to(torch.bfloat16).to(DEV)
        o = torch.empty(T, d, dtype=torch.bfloat16, device=DEV)
        dec.pos.fill_(n)
        dec._attend_few(0, rows, o)
        n += T
        k, v = (x.cpu().double().transpose(1, 2) for x in ops.kv8_read(dec.caches[0], torch.tensor([n], dtype=torch.int32, device=DEV), n))
        q = rows.view(1, T, 3, H, hd)[:, :, 0].cpu()
        want, absv, big = attention(q, k, v, [n - T], [T], [0], 0, 0, hd ** -0.5, torch.zeros(1, T, H, hd))
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -16 + 2 * hd * 2.0 ** -23 * big + 96 * 2.0 ** -23 + 2.0 ** -21) * absv
        assert bool(((o.view(1, T, H, hd).cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("kind,gate", [("int8", 5e-2), ("e4m3", 1e-1)])
def test_predict_text_8bit(kind, gate, monkeypatch):
    """Decoding from an 8-bit cache stays near the bf16 one (int8: a code is off by at most amax / 127 of its block, e4m3: 2^-4 of its value, both
    averaged by the softmax and added to the residual stream), replayed graph and eager steps agree, calls repeat."""
    m = _policy(layers=2)
    want, _ = m.predict_text(_prompt(30), max_length=1)
    m.kv_cache = kind
    got, _ = m.predict_text(_prompt(30), max_length=1)
    assert float((got - want).abs().max()) < gate * float(want.abs().max())
    monkeypatch.setenv("NEKO_DECODE_GRAPH", "1")
    l1, t1 = m.predict_text(_prompt(30), max_length=12)
    l2, t2 = m.predict_text(_prompt(30), max_length=12)
    monkeypatch.setenv("NEKO_DECODE_GRAPH", "0")
    l3, t3 = m.predict_text(_prompt(30), max_length=12)
    assert torch.equal(l1, l2) and [int(t) for t in t1] == [int(t) for t in t2] == [int(t) for t in t3]
    assert float((l1 - l3).abs().max()) < 2e-2 * float(l3.abs().max())


def test_windowed_decode_runs_past_the_context():
    """decode_window: a sequence outgrows context_len without being recomputed; a window that covers everything changes nothing; bf16 refuses."""
    m = _policy(ctx=64)
    m.kv_cache = "int8"
    plain, _ = m.predict_text(_prompt(20), max_length=30)
    m.decode_window = 64
    same, _ = m.predict_text(_prompt(20), max_length=30)
    assert torch.equal(plain, same)
    m.decode_window, m.decode_sinks = 16, 4
    l, t = m.predict_text(_prompt(50), max_length=60)
    assert l.shape[0] == 60 and len(t) == 60 and bool(torch.isfinite(l).all())
    m.kv_cache = "bf16"
    with pytest.raises(ValueError, match="decode_window"):
        m.predict_text(_prompt(20), max_length=2)
    m.decode_window, m.kv_cache = 0, "fp4"
    with pytest.raises(ValueError, match="kv_cache"):
        m.predict_text(_prompt(20), max_length=2)


@pytest.mark.parametrize("kind", ["bf16", "int8", "e4m3"])
@pytest.mark.parametrize("n_draft", [1, 4, 7])
@pytest.mark.parametrize("same", [True, False])
def test_speculative_greedy(kind, n_draft, same):
    """Greedy drafted decoding emits the argmax of the logits it returns, whoever drafts, and those logits are the policy's own: a plain decode forced
    along the same tokens gives them within the caches' rounding."""
    m = _policy(seed=0)
    draft = m if same else _policy(seed=3, layers=1)
    m.kv_cache = draft.kv_cache = kind
    p = _prompt(25)
    logits, tokens = m.predict_text_speculative(p, draft, max_length=15, n_draft=n_draft)
    ids = [int(t) for t in tokens]
    assert logits.shape[0] == 15 and ids == logits.argmax(-1).tolist()
    dec = m._new_decoder(m.context_len, torch.device(DEV))
    from neko_amd import engine
    table, hp = m._flat.view("embed_token.weight"), m._head_params()
    h = dec.extend(m.tokenize_input_dicts([p])[0][0].float())
    for i, t in enumerate(ids):
        lg = engine.lm_head_rows(hp, h[-1:])[0, :128]
        assert float((lg - logits[i]).abs().max()) < {"bf16": 2e-2, "int8": 5e-2, "e4m3": 1e-1}[kind] * float(lg.abs().max())
        h = dec.extend(table[t].reshape(1, -1))


def test_speculative_sampled_and_refusals():
    m, draft = _policy(seed=0), _policy(seed=5, layers=1)
    m.kv_cache = "int8"
    gen = torch.Generator(device=DEV)
    outs = []
    for _ in range(2):
        gen.manual_seed(7)
        l, t = m.predict_text_speculative(_prompt(20), draft, max_length=12, deterministic=False, temperature=0.9, generator=gen)
        assert l.shape[0] == 12 and all(0 <= int(x) < 128 for x in t)
        outs.append([int(x) for x in t])
    assert outs[0] == outs[1]
    for bad in (dict(n_draft=0), dict(n_draft=8), dict(max_length=200), dict(deterministic=False, temperature=0.0)):
        with pytest.raises(ValueError):
            m.predict_text_speculative(_prompt(20), draft, **bad)
    from neko_amd.policy.gato_policy import GatoPolicy
    other = GatoPolicy(DEV, 64, 1, 2, 0.0, resid_mid_channels=128, context_len=96, text_tokenizer=64)
    with pytest.raises(ValueError, match="vocabulary"):
        m.predict_text_speculative(_prompt(20), other)


def _batch():
    g = torch.Generator().manual_seed(2)
    return [{"text": torch.randint(0, 128, (21,), generator=g).tolist()},
            {"continuous_obs": torch.randn(4, 5, generator=g).to(DEV), "continuous_actions": (torch.rand(4, 2, generator=g) * 2 - 1).to(DEV)}]


def _grads(m, teacher):
    m._flat.zero_grad()
    _, loss = m.forward(_batch(), compute_loss=True, return_logits=False, teacher=teacher)
    loss.backward()
    torch.cuda.synchronize()
    return float(loss), {n: p.grad.detach().clone() for n, p in m.named_parameters() if p.grad is not None}


def test_distillation_step():
    """A student's loss and gradients under a teacher: hard = 1 is the ordinary step, hard = 0 the definition on the student's own logits, and a mixture
    the mixture of the two.  (The backward is linear in the logits' gradient but for its bf16 roundings: about eight on the way to a weight, in
    each of the three runs, 2^-9 rms each -> 24 x 0.58 x 2^-9 < 2^-5 of the terms' norms.)"""
    from neko_amd import engine
    teacher_policy, m = _policy(seed=9, d=128), _policy(seed=0)
    t = teacher_policy.top_logits(_batch(), 16, tau=2.0)
    n = t.values.shape[0]
    logits, plain_loss = m.forward(_batch(), compute_loss=True)
    rows = logits.view(-1, m.vocab_size)[m.last_pack.loss_idx[:n].long()].detach().cpu().to(torch.bfloat16)
    l_ce, g_ce = _grads(m, None)
    l_hard, g_hard = _grads(m, engine.Teacher(t.values, t.indices, 2.0, 1.0))
    assert abs(l_hard - l_ce) < 1e-5 * abs(l_ce)
    for k in g_ce:
        assert float((g_hard[k] - g_ce[k]).abs().max()) <= 2e-2 * float(g_ce[k].abs().max()) + 1e-12, k
    l_soft, g_soft = _grads(m, t)
    want, _, _ = distill(rows, m.vocab_size, t.values.cpu(), t.indices.cpu(), torch.full((n,), 1.0 / n), 2.0, None, 0.0)
    assert abs(l_soft - float(want.mean())) < 1e-3 * abs(float(want.mean()))
    l_mix, g_mix = _grads(m, engine.Teacher(t.values, t.indices, 2.0, 0.25))
    assert abs(l_mix - (0.75 * l_soft + 0.25 * l_ce)) < 1e-5 * abs(l_mix)
    for k in g_mix:
        ref = 0.75 * g_soft[k] + 0.25 * g_ce[k]
        assert float((g_mix[k] - ref).norm()) <= 2.0 ** -5 * float((0.75 * g_soft[k]).norm() + (0.25 * g_ce[k]).norm()) + 1e-12, k


def test_distillation_refusals():
    m = _policy(seed=0)
    t = m.top_logits(_batch(), 4)
    from neko_amd import engine
    with pytest.raises(ValueError, match="loss rows"):
        m.forward(_batch(), compute_loss=True, teacher=engine.Teacher(t.values[:-1], t.indices[:-1]))
    with pytest.raises(ValueError, match="compute_loss"):
        m.forward(_batch(), teacher=t)


def test_speculative_ends_on_logits_that_are_no_numbers():
    m, draft = _policy(seed=0), _policy(seed=5, layers=1)
    with torch.no_grad():
        dict(m.named_parameters())["predict_token.weight"].fill_(float("nan"))
    m._flat.ensure_shadow()
    with pytest.raises(RuntimeError, match="no number"):
        m.predict_text_speculative(_prompt(20), draft, max_length=4)
    with pytest.raises(ValueError, match="max_length"):
        m.predict_text_speculative(_prompt(20), draft, max_length=0)
