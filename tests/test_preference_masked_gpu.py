"""The preference loss where a token of an answer is masked (logit -inf): its answer is
infinitely unlikely, and the pair's loss and coefficient are their limits."""
import math

import pytest

import tensorplay_amd as tp
from tests import finetune_util as F
from tests.test_logits_losses_gpu import DTYPES, _stream, make  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("eps", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("masked", ["other", "preferred", "both"])
def test_masked_token(masked, eps, dtype):
    print(f"case masked {masked} eps={eps} {dtype}", flush=True)
    x, t, g = make(12, 300, dtype, 40)
    cut = torch.tensor([0, 3, 6, 9, 12], device="cuda")   # pair 0: rows 0-2 and 6-8, pair 1: 3-5 and 9-11
    for row in {"other": [7], "preferred": [1], "both": [1, 7]}[masked]:
        x[row, int(t[row])] = -math.inf
    f, beta, inf = tp.from_torch, 0.4, math.inf
    ref = torch.randn((4,), generator=g, device="cuda")
    loss, reward, logp, lse, coef = tp.preference_loss(f(x), f(t), f(cut), f(ref), beta, eps)
    one = torch.ones((), device="cuda")
    grad = tp.to_torch(tp.preference_loss_backward(f(one), coef, f(x), f(t), lse))
    loss, reward, logp, coef = (tp.to_torch(v) for v in (loss, reward, logp, coef))
    want, p, tol = F.logprob64(x, t)
    F.assert_within(logp, want, tol, "logp")
    assert reward[0].item() == -inf if masked != "other" else math.isfinite(reward[0])
    assert reward[2].item() == -inf if masked != "preferred" else math.isfinite(reward[2])
    if masked == "both":     # neither can be told from the other
        assert math.isnan(loss) and bool(coef[[0, 1, 2, 6, 7, 8]].isnan().all())
    else:
        # h = inf: down = 0, up = 1; h = -inf the other way round
        h_up, h_down = (1.0, 0.0) if masked == "other" else (0.0, 1.0)
        c = beta / 2 * (eps * h_up - (1 - eps) * h_down)
        r = torch.full((6,), c, dtype=torch.float64, device="cuda")
        c64 = torch.cat([r[:3], coef[3:6].double(), -r[3:], coef[9:].double()])
        F.assert_within(coef, c64, 2 * F.U * c64.abs(), "coef")
        finite = (eps if masked == "other" else 1 - eps) == 0
        assert math.isfinite(loss) if finite else loss.item() == inf
        if finite:           # what is left is the other pair's, whose sigmoid moves with its tokens' error
            h = beta * float(want[3:6].sum() - ref[1].double() - want[9:].sum() + ref[3].double())
            sig = lambda v: math.log1p(math.exp(v))
            l64 = ((1 - eps) * sig(-h) + eps * sig(h)) / 2
            assert abs(float(loss) - l64) <= beta * float(tol[[3, 4, 5, 9, 10, 11]].sum()) + 4 * F.U * l64
        ls = F.stats64(x, 1.0)[1]
        gref = F.logits_grad64(c64, want, p, t, 1.0)
        F.assert_within(grad, gref, F.logits_grad_tol(c64, want, p, ls, 1.0, dtype, tol, gref), "grad")
    # the pair that is not masked is as it would be without the other
    rows = [3, 4, 5, 9, 10, 11]
    assert bool(coef[rows].isfinite().all()) and bool(grad[rows].isfinite().all())
