"""The preference loss of pairs that are far apart: losses and coefficients of e^-h and
less keep their digits."""
import math

import pytest

import tensorplay_amd as tp
from tests import finetune_util as F
from tests.test_logits_losses_gpu import DTYPES, _stream, make  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def pairs_apart(hs, lens, vocab, dtype, beta, seed):
    """A pair for each h, of lens[0] preferred and lens[1] other tokens, whose rewards
    differ by about h: the reference sums make up the rest."""
    n = len(hs)
    x, t, g = make(n * sum(lens), vocab, dtype, seed)
    cut = torch.tensor([0] + [lens[i >= n] for i in range(2 * n)], device="cuda").cumsum(0)
    want, p, tol = F.logprob64(x, t)
    sums = torch.stack([want[int(a):int(b)].sum() for a, b in zip(cut, cut[1:])])
    half = torch.tensor(hs, dtype=torch.float64, device="cuda") / 2 / beta
    return x, t, cut, (sums - torch.cat([half, -half])).float()


def check_separated(x, t, cut, ref, beta, eps):
    f, pairs = tp.from_torch, (len(cut) - 1) // 2
    loss, reward, logp, lse, coef = tp.preference_loss(f(x), f(t), f(cut), f(ref), beta, eps)
    scale = torch.tensor(2.0, device="cuda")
    grad = tp.to_torch(tp.preference_loss_backward(f(scale), coef, f(x), f(t), lse))
    want, p, tol = F.logprob64(x, t)
    seq = [slice(int(a), int(b)) for a, b in zip(cut, cut[1:])]
    # a reward: its tokens' errors and the roundings of 64-bit sums, which U covers by far
    sums = torch.stack([want[s].sum() for s in seq])
    stol = torch.stack([tol[s].sum() for s in seq]) * beta + F.U / 1024 * beta * (sums.abs() + ref.double().abs())
    r = beta * (sums - ref.double())
    h, htol = r[:pairs] - r[pairs:], stol[:pairs] + stol[pairs:]
    up, down = torch.sigmoid(h), torch.sigmoid(-h)
    sig = torch.nn.functional.logsigmoid
    part = -(1 - eps) * sig(h) - eps * sig(-h)
    dh = (eps * up - (1 - eps) * down) * beta / pairs
    # sigmoids move by e^htol at most where h moves by htol, the loss by their sum, the
    # coefficient by their product; one rounding to 32 bits after 64-bit arithmetic
    grow = htol.exp() * htol
    ltol = float((grow * (eps * up + (1 - eps) * down)).mean()) + 2 * F.U * float(part.mean())
    dtol = grow * up * down * beta / pairs + 2 * F.U * dh.abs() + 2.0 ** -126
    c64, ctol = torch.zeros_like(want), torch.zeros_like(want)
    for i, s in enumerate(seq):
        c64[s], ctol[s] = dh[i % pairs] * (1 if i < pairs else -1), dtol[i % pairs]
    F.assert_within(tp.to_torch(logp), want, tol, "logp")
    F.assert_within(tp.to_torch(reward), r, stol + F.U * r.abs(), "reward")
    F.assert_within(tp.to_torch(loss), part.mean(), ltol, "loss")
    F.assert_within(tp.to_torch(coef), c64, ctol, "coef")
    ls = F.stats64(x, 1.0)[1]
    gref = F.logits_grad64(c64 * 2, want, p, t, 1.0)
    at = torch.zeros_like(p).scatter_(1, t[:, None], 1.0)
    gtol = F.logits_grad_tol(c64 * 2, want, p, ls, 1.0, x.dtype, tol, gref) + 2 * ctol[:, None] * torch.maximum(p, at)
    F.assert_within(grad, gref, gtol, "grad")


@pytest.mark.parametrize("eps", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("h", [20.0, -20.0, 40.0, -40.0, 80.0, -80.0, 0.5])
def test_one_pair(h, eps):
    for dtype in DTYPES:
        print(f"case pair h={h} eps={eps} {dtype}", flush=True)
        check_separated(*pairs_apart([h], (7, 4), 501, dtype, 0.5, 30), 0.5, eps)


@pytest.mark.parametrize("eps", [0.0, 0.1])
def test_pairs_in_one_and_in_several_launches(eps):
    hs = [30.0 * math.sin(i) for i in range(40)]
    check_separated(*pairs_apart(hs, (3, 5), 130, torch.bfloat16, 0.3, 31), 0.3, eps)
    # all of them far apart, so that no near pair hides the loss; more than 16384 tokens
    hs = [25.0 + (i * 37 % 101) / 10 for i in range(1100)]
    check_separated(*pairs_apart(hs, (7, 9), 12, torch.float32, 1.0, 32), 1.0, eps)
