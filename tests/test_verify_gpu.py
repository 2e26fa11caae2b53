"""Verification of drafted tokens against a 64-bit restatement: whole numbers, equal."""
import math

import pytest
import torch

from serving_ref import verify

pytestmark = pytest.mark.gpu


def _case(B, K, V, temperature, with_draft, dtype, seed, ld=0, sharp=2.0):
    g = torch.Generator().manual_seed(seed)
    ld = max(ld, V)
    t = torch.randn(B, K + 1, ld, generator=g).mul(sharp).to(dtype)
    d = (t[:, :K].float() + 0.5 * torch.randn(B, K, ld, generator=g)).to(dtype)
    x = torch.distributions.Categorical(logits=d[:, :, :V].float() / max(temperature, 0.3)).sample() if with_draft else t[:, :K, :V].float().argmax(-1)
    x = torch.where(torch.rand(B, K, generator=g) < 0.15, torch.randint(0, V, (B, K), generator=g), x)
    u, r = torch.rand(B, K, generator=g), torch.rand(B, generator=g)
    n = torch.randint(0, K + 1, (B,), generator=g).to(torch.int32)
    n[0] = K
    return t[:, :, :V], x, (d[:, :, :V] if with_draft else None), u, r, n


def _run(t, x, d, u, r, n, temperature):
    from neko_amd import ops
    dev = lambda a: None if a is None else a.cuda()

    def rows(a):       # keep the row padding on the device
        if a is None:
            return None
        base = torch.zeros(a.shape[0], a.shape[1], a.stride(1), dtype=a.dtype, device="cuda")
        base[:, :, :a.shape[2]] = a.cuda()
        return base[:, :, :a.shape[2]]
    acc, out = ops.verify_draft(rows(t), dev(x), draft_logits=rows(d), u=dev(u), r=dev(r), n_draft=dev(n), temperature=temperature)
    return acc.tolist(), out.tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0, 3.0])
@pytest.mark.parametrize("B,K,V,ld", [(1, 1, 1, 0), (3, 2, 7, 9), (9, 5, 4096, 0), (4, 4, 4097, 4160), (5, 8, 52305, 52480), (2, 62, 300, 0)])
def test_verify(B, K, V, ld, temperature, with_draft, dtype):
    c = _case(B, K, V, temperature, with_draft, dtype, seed=B * 100 + K, ld=ld)
    assert _run(*c, temperature) == verify(*c, temperature)


def test_verify_many_borders():
    """Flat distributions over the whole vocabulary: the border falls between neighbours 2e-5 apart, a hundred times."""
    c = _case(100, 1, 52305, 1.0, True, torch.float32, seed=4, sharp=0.05)
    assert _run(*c, 1.0) == verify(*c, 1.0)


def test_verify_special_rows():
    """Masked logits (-inf), NaN, +inf, rows without any finite logit, tokens outside the vocabulary, equal distributions, r at its ends."""
    B, K, V = 8, 3, 130
    t, x, d, u, r, n = _case(B, K, V, 1.0, True, torch.float32, seed=2)
    t, d = t.clone(), d.clone()
    n[:] = K
    t[0, :, 5:] = -math.inf                      # five tokens left
    t[1, 0] = -math.inf                          # nothing to sample
    t[2, 1, 7] = math.nan
    t[2, 0, 9] = math.inf
    t[3, 0, [3, 99]] = math.inf                  # two infinite logits share the mass
    d[4] = t[4, :K]                              # equal: everything is kept
    x[5, 0], x[6, 0] = -1, V
    t[7, :, 1:] = -math.inf                      # one token
    r[0], r[3] = 0.0, 0.99999994
    u[4] = 0.99999994
    for temperature in (1.0, 0.0, 0.5):
        for draft in (d, None):
            c = (t, x, draft, u, r, n, temperature)
            if draft is not None and temperature == 1.0:
                assert verify(*c)[0][4] == K
            assert _run(*c) == verify(*c), (temperature, draft is None)


def test_verify_ties_greedy():
    t = torch.zeros(2, 3, 9000)
    t[0, 0, [17, 5000, 8999]] = 2.0
    t[1] = 1.0
    x = torch.tensor([[17, 0], [0, 1]])
    n = torch.tensor([2, 2], dtype=torch.int32)
    assert _run(t, x, None, None, None, n, 0.0) == ([2, 1], [[17, 0, 0], [0, 0, -1]])


def test_verify_captured():
    from neko_amd import ops
    c = _case(4, 3, 1000, 1.0, True, torch.float32, seed=8)
    t, x, d, u, r, n = (a.cuda() for a in c)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        acc, out = ops.verify_draft(t, x, draft_logits=d, u=u, r=r, n_draft=n)
    for seed in range(3):
        gen = torch.Generator().manual_seed(seed)
        u2, r2 = torch.rand(c[3].shape, generator=gen), torch.rand(c[4].shape, generator=gen)
        u.copy_(u2)
        r.copy_(r2)
        g.replay()
        torch.cuda.synchronize()
        assert (acc.tolist(), out.tolist()) == verify(c[0], c[1], c[2], u2, r2, c[5], 1.0)
        eager = ops.verify_draft(t, x, draft_logits=d, u=u, r=r, n_draft=n)
        assert torch.equal(eager[0], acc) and torch.equal(eager[1], out)


def test_verify_keeps_the_target_distribution():
    """The law of speculative sampling on a 4-token vocabulary: the first token out follows the target's softmax, whatever the draft proposed.
    4 sigma of a frequency over N independent rows."""
    from neko_amd import ops
    N, V = 20000, 4
    g = torch.Generator().manual_seed(0)
    t = torch.tensor([0.3, -1.0, 1.2, 0.0])
    d = torch.tensor([1.0, 0.5, -0.5, 0.2])
    x = torch.multinomial(torch.softmax(d, 0), N, replacement=True, generator=g).reshape(N, 1)
    u, r = torch.rand(N, 1, generator=g), torch.rand(N, generator=g)
    _, out = ops.verify_draft(t.expand(N, 2, V).contiguous().cuda(), x.cuda(), draft_logits=d.expand(N, 1, V).contiguous().cuda(), u=u.cuda(), r=r.cuda())
    freq = torch.bincount(out[:, 0].cpu(), minlength=V).double() / N
    p = torch.softmax(t.double(), 0)
    assert bool(((freq - p).abs() <= 4 * (p * (1 - p) / N).sqrt()).all()), (freq, p)


@pytest.mark.parametrize("temperature", [1e-3, 1e-12, 1e-30])
@pytest.mark.parametrize("with_draft", [True, False])
def test_verify_cold(temperature, with_draft):
    """Temperatures next to zero: the largest logit has all the mass, in every piece of the row, whatever logit / temperature comes to."""
    t, x, d, u, r, n = _case(6, 4, 9001, 1.0, with_draft, torch.float32, seed=8)
    x[:4] = t[:4, :4].argmax(-1)
    c = (t, x, d, u, r, n)
    assert _run(*c, temperature) == verify(*c, temperature)
