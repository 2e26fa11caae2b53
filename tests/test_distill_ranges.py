"""Distillation at temperatures from the smallest normal number on, and sums as deep as the vocabulary makes them."""
import math

import pytest
import torch

from neko_amd import _lib
from serving_ref import distill
from test_distill_gpu import _case, _run
from test_serving_refusals_cpu import DISTILL


@pytest.mark.parametrize("tau", [math.inf, -math.inf, 1e-39, -1.0])
def test_refused_temperatures(tau):
    assert _lib.load().neko_distill_topk(*{**DISTILL, "tau": tau}.values()) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tau", [1e-15, 1e-20, 1e-25, 1e-30, 1.2e-38])
def test_very_cold(tau, dtype):
    """Both distributions are one token: the loss is tau times the gap between the two logits, though tau^2 is below fp32 and a gap / tau above it."""
    R, V, k = 3, 2000, 4
    z, Vpad, tv, ti, w, y = _case(R, V, k, dtype, seed=2)
    best = torch.tensor([5, 900, 1999])
    z[torch.arange(R), best] = 20.0
    tv[:, 1] = 50.0
    loss, dz = _run(z, V, Vpad, tv, ti, w, y, tau, 0.0)
    t32 = float(torch.tensor(tau, dtype=torch.float32))
    for r in range(R):
        t, s = int(ti[r, 1]), int(best[r])
        gap = t32 * (20.0 - float(z[r, t]))
        assert abs(float(loss[r]) - gap) <= 4 * 2.0 ** -24 * gap           # the difference, its product with t = 1, two products
        want = torch.zeros(V, dtype=torch.float64)
        want[s] += float(w[r]) * t32
        want[t] -= float(w[r]) * t32
        # bf16: the stored rounding, and the factor's logarithm (below 128 in size: half a step is 2^-18; a second one for the logarithm) in the exponent;
        # fp32: four products and the exponential; and results below the smallest normal number may be 0
        rel = 2.0 ** -8 + 2.0 ** -17 if dtype == torch.bfloat16 else 4 * 2.0 ** -24 + 2.0 ** -22
        assert bool(((dz[r, :V].double() - want).abs() <= rel * want.abs() + 2.0 ** -126).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [52305, 106000, 150000, 400000])
@pytest.mark.parametrize("tau,hard", [(2.5, 0.0), (2.0, 0.3), (1.0, 1.0)])
def test_long_rows(V, tau, hard, dtype):
    """The tolerance's depth from the row: a thread of 512 or 1024 adds its terms one after the other, then lanes and waves meet."""
    R, k = 2, 20
    z, Vpad, tv, ti, w, y = _case(R, V, k, dtype, seed=V)
    loss, dz = _run(z, V, Vpad, tv, ti, w, y, tau, hard)
    rl, rg, mag = distill(z, V, tv, ti, w, tau, y, hard)
    per = 8 if dtype == torch.bfloat16 else 4
    depth = -(-V // (512 * per)) * per + 6 + 16                            # 512 threads at least; six levels of a wave, the waves' 16 sums
    x = z[:, :V].float()
    span = float((x.amax(1) - x.amin(1)).max()) + 1
    # an exponent's argument: the difference, the constant, their product (half a step each, of up to span / tau log2 e); the exponential 2^-21
    rel = 2 * depth * 2.0 ** -24 + 3 * span * 1.45 / min(tau, 1.0) * 2.0 ** -24 + 2.0 ** -21
    size = (1 - hard) * tau * tau * (span / tau + math.log(V) + math.log(k) + 1) + hard * (span + math.log(V) + 1)
    assert bool(((loss.double() - rl).abs() <= 2 * (rel + 8 * 2.0 ** -24) * size).all())
    out_round = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    fold = 2.0 ** -18 if dtype == torch.bfloat16 else 0.0                  # the folded factor's logarithm in the exponent (below 64 in size)
    assert bool(((dz[:, :V].double() - rg).abs() <= out_round * rg.abs() + (2 * rel + fold) * mag + 1e-38).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_single_row_of_any_width(dtype):
    """One row beside others' columns: there is no stride to be a multiple of 16 bytes, and columns behind Vpad stay."""
    from neko_amd import ops
    z, Vpad, tv, ti, w, y = _case(1, 300, 5, dtype, seed=1)
    loss, dz = _run(z, 300, Vpad, tv, ti, w, y, 2.0, 0.3)
    for extra in (1, 3, 16):
        wide = torch.full((1, Vpad + extra), 5.0, dtype=dtype, device="cuda")
        wide[:, :Vpad] = z.cuda()
        out, l2 = torch.full_like(wide, 7.0), torch.empty(1, device="cuda")
        ops.distill_topk(wide, 300, Vpad, tv.cuda(), ti.cuda(), w.cuda(), tau=2.0, target=y.cuda(), hard=0.3, loss_row=l2, dlogits=out)
        assert torch.equal(l2.cpu(), loss) and torch.equal(out[:, :Vpad].cpu(), dz) and bool((out[:, Vpad:] == 7).all())
