"""Distillation from a teacher's top logits: loss and gradient against a 64-bit restatement and against differences."""
import math

import pytest
import torch

from serving_ref import distill

pytestmark = pytest.mark.gpu


def _case(R, V, k, dtype, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    n = 8 if dtype == torch.bfloat16 else 4
    Vpad = (V + n - 1) // n * n + pad
    z = torch.full((R, Vpad), float("nan"), dtype=dtype)          # padding columns are never looked at
    z[:, :V] = (torch.randn(R, V, generator=g) * 2).to(dtype)
    tv = torch.randn(R, k, generator=g) * 3
    ti = torch.stack([torch.randperm(V, generator=g)[:k] if V >= k else torch.randint(0, V, (k,), generator=g) for _ in range(R)]).to(torch.int32)
    w = torch.rand(R, generator=g) + 0.1
    y = torch.randint(0, V, (R,), generator=g)
    return z, Vpad, tv, ti, w, y


def _run(z, V, Vpad, tv, ti, w, y, tau, hard, inplace=False):
    from neko_amd import ops
    zd = z.cuda()
    loss = torch.empty(z.shape[0], device="cuda")
    dz = zd if inplace else torch.full_like(zd, 3.0)
    ops.distill_topk(zd, V, Vpad, tv.cuda() if tv is not None else None, ti.cuda() if ti is not None else None, w.cuda(), tau=tau,
                     target=y.cuda() if y is not None else None, hard=hard, loss_row=loss, dlogits=dz)
    return loss.cpu(), dz.cpu()


def _check(z, V, Vpad, tv, ti, w, y, tau, hard, inplace=False):
    loss, dz = _run(z, V, Vpad, tv, ti, w, y, tau, hard, inplace)
    rl, rg, mag = distill(z, V, tv, ti, w, tau, y, hard)
    # an exponential's argument (z - m) / tau, |z - m| <= span, is off by 2 roundings of it, its value by 2^-21 more; a sum of V positive
    # terms in a tree of at most 96 levels by 96 roundings; a logarithm and the loss's few terms, each at most span + ln V, by 8 more
    span = float((z[:, :V].float().nan_to_num(neginf=0).amax(1) - z[:, :V].float().nan_to_num(neginf=0).amin(1)).max()) + 1
    rel = (2 * span * 1.45 / min(tau, 1.0) + 8 + 96) * 2.0 ** -23
    size = (1 - hard) * tau * tau * (span / tau + math.log(V) + math.log(max(1, ti.shape[1] if ti is not None else 1)) + 1) + hard * (span + math.log(V) + 1)
    fin = torch.isfinite(rl)
    assert torch.equal(torch.isfinite(loss), fin)
    assert bool(((loss.double() - rl).abs()[fin] <= (rel + 8 * 2.0 ** -24) * size * 2).all()), float((loss.double() - rl).abs()[fin].max())
    out_round = 2.0 ** -8 if z.dtype == torch.bfloat16 else 2.0 ** -24
    err = (dz[:, :V].double() - rg).abs()
    assert bool((err <= out_round * rg.abs() + 2 * rel * mag + 1e-38).all()), float((err - out_round * rg.abs() - 2 * rel * mag).max())
    assert int(dz[:, V:Vpad].count_nonzero()) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,k", [(1, 1), (33, 5), (1000, 64), (2048, 1), (5000, 130), (30000, 16), (52305, 64), (120001, 32)])
@pytest.mark.parametrize("tau,hard", [(1.0, 0.0), (2.5, 0.3), (1.0, 0.5), (0.7, 1.0)])
def test_distill(V, k, tau, hard, dtype):
    R = 3
    z, Vpad, tv, ti, w, y = _case(R, V, k, dtype, seed=V + k)
    _check(z, V, Vpad, tv, ti, w, y, tau, hard)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [700, 20000, 52305, 150000])
def test_distill_in_place_and_padding(V, dtype):
    z, Vpad, tv, ti, w, y = _case(4, V, 20, dtype, seed=V, pad=64)
    _check(z, V, Vpad, tv, ti, w, y, 1.5, 0.25, inplace=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_distill_edges(dtype):
    """Equal indices, the label among them, entries that are none, a row without a teacher, without a label, weight 0, masked student logits."""
    V, k = 300, 6
    z, Vpad, tv, ti, w, y = _case(7, V, k, dtype, seed=1)
    ti[0] = torch.tensor([5, 5, 9, 5, 9, 7])
    y[0] = 5
    ti[1, 2:] = torch.tensor([-1, V, 2 ** 31 - 1, -2 ** 31])
    tv[2] = -math.inf                              # no teacher
    y[3] = -100                                    # no label
    w[4] = 0.0
    ti[5], tv[5] = -1, 1.0
    y[5] = -1                                      # neither
    z[6, 100:200] = -math.inf
    ti[6] = torch.tensor([1, 2, 3, 4, 250, 299])
    y[6] = 7
    for tau, hard in ((1.0, 0.0), (2.0, 0.4), (3.0, 1.0)):
        _check(z, V, Vpad, tv, ti, w, y, tau, hard)
        loss, dz = _run(z, V, Vpad, tv, ti, w, y, tau, hard)
        assert float(loss[4]) == 0 and int(dz[4].count_nonzero()) == 0
        assert float(loss[5]) == 0 and int(dz[5].count_nonzero()) == 0


def test_distill_gradient_against_differences():
    """d(sum w loss)/dz in fp32 against central differences of the 64-bit loss (step h: truncation h^2/6 times a third derivative below 2 / tau)."""
    V, k, R, tau, hard, h = 40, 7, 2, 1.7, 0.35, 1e-4
    z, Vpad, tv, ti, w, y = _case(R, V, k, torch.float32, seed=3)
    _, dz = _run(z, V, Vpad, tv, ti, w, y, tau, hard)
    for r in range(R):
        for c in range(V):
            up, dn = z.double().clone(), z.double().clone()
            up[r, c] += h
            dn[r, c] -= h
            a = distill(up, V, tv, ti, w, tau, y, hard)[0][r]
            b = distill(dn, V, tv, ti, w, tau, y, hard)[0][r]
            assert abs(float(w[r]) * float(a - b) / (2 * h) - float(dz[r, c])) < 1e-5


def test_distill_matches_cross_entropy_kernel():
    """hard = 1 is the framework's masked cross-entropy: same loss and gradient to a rounding."""
    from neko_amd import ops
    R, V = 5, 52305
    z, Vpad, _, _, w, y = _case(R, V, 1, torch.bfloat16, seed=11)
    z = z.nan_to_num(0.0)
    loss, dz = _run(z, V, Vpad, None, None, w, y, 1.0, 1.0)
    zc = z.cuda()
    lc = torch.empty(R, device="cuda")
    ops.ce_bf16_inplace(zc, V, Vpad, y.cuda(), w.cuda(), loss_row=lc)
    assert float((loss - lc.cpu()).abs().max()) <= 110 * 2.0 ** -23 * 30
    assert bool(((dz.float() - zc.cpu().float()).abs() <= 2.0 ** -7 * dz.float().abs() + 1e-8).all())


def test_distill_captured_and_loss_only():
    from neko_amd import ops
    V, k = 2000, 8
    z, Vpad, tv, ti, w, y = (a.cuda() if torch.is_tensor(a) else a for a in _case(6, V, k, torch.float32, seed=5))
    loss, dz = torch.empty(6, device="cuda"), torch.empty_like(z)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        ops.distill_topk(z, V, Vpad, tv, ti, w, tau=2.0, loss_row=loss, dlogits=dz)
    for i in range(3):
        z[:, :V].normal_()
        g.replay()
        torch.cuda.synchronize()
        l2, d2, l3 = torch.empty_like(loss), torch.empty_like(dz), torch.empty_like(loss)
        ops.distill_topk(z, V, Vpad, tv, ti, w, tau=2.0, loss_row=l2, dlogits=d2)
        ops.distill_topk(z, V, Vpad, tv, ti, w, tau=2.0, loss_row=l3)
        assert torch.equal(loss, l2) and torch.equal(dz, d2) and torch.equal(l2, l3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [300, 30000, 120001])
def test_distill_lowest_values(V, dtype):
    """Logits of the type's lowest value: a row that holds nothing else is a flat one, and beside ordinary logits they count as -inf."""
    z, Vpad, tv, ti, w, y = _case(3, V, 6, dtype, seed=V)
    low = torch.finfo(dtype).min
    flat = z.clone()
    flat[:, :V] = low
    for tau, hard in ((1.0, 0.0), (2.0, 0.4), (0.5, 1.0)):
        _check(flat, V, Vpad, tv, ti, w, y, tau, hard)
    ti = ti % 50
    y = y % 50
    a, b = z.clone(), z.clone()
    a[:, 50:V], b[:, 50:V] = low, -math.inf
    for tau, hard in ((1.0, 0.0), (2.0, 0.4), (0.5, 1.0)):
        got, want = _run(a, V, Vpad, tv, ti, w, y, tau, hard), _run(b, V, Vpad, tv, ti, w, y, tau, hard)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert bool(torch.isfinite(got[0]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tau", [1e-6, 1e-12])
def test_distill_cold(tau, dtype):
    """tau next to zero: both distributions are one token, the loss is tau times the gap between them."""
    R, V, k = 3, 2000, 4
    z, Vpad, tv, ti, w, y = _case(R, V, k, dtype, seed=2)
    best = torch.tensor([5, 900, 1999])
    z[torch.arange(R), best] = 20.0
    tv[:, 1] = 50.0
    loss, dz = _run(z, V, Vpad, tv, ti, w, y, tau, 0.0)
    for r in range(R):
        t, s = int(ti[r, 1]), int(best[r])
        gap = tau * (20.0 - float(z[r, t]))
        # half a step of fp32 each: tau, log2(e), their quotient, the difference, its product with it, ln 2, the product with that, (1 - hard) tau tau
        # in two products, and the last one
        assert abs(float(loss[r]) - gap) <= 10 * 2.0 ** -24 * gap
        want = torch.zeros(V, dtype=torch.float64)
        want[s] += float(w[r]) * tau
        want[t] -= float(w[r]) * tau
        # bf16: the stored rounding, and the factor's logarithm (below 64 in size: half a step is 2^-19; a second one for the logarithm itself)
        # in the exponent; fp32: four products
        rel = 2.0 ** -8 + 2.0 ** -18 if dtype == torch.bfloat16 else 4 * 2.0 ** -24 + 2.0 ** -22
        assert bool(((dz[r, :V].double() - want).abs() <= rel * want.abs()).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hard", [0.0, 0.4])
@pytest.mark.parametrize("pieces", [257, 513, 1300, 2100, 3100, 4097, 4700, 5500, 6100, 7100, 7700, 9001, 11000])
def test_distill_every_row_length(pieces, hard, dtype):
    """Rows of that many 16-byte pieces, the last one partly filled: one per number of rounds a row can take."""
    n = 8 if dtype == torch.bfloat16 else 4
    V = pieces * n - 3
    z, Vpad, tv, ti, w, y = _case(2, V, 9, dtype, seed=pieces)
    assert Vpad == pieces * n
    _check(z, V, Vpad, tv, ti, w, y, 2.0, hard)
