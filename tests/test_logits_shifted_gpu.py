"""Log-probabilities and the policy loss do not change when all logits of a row move by a
constant: rows far from 0, and rows whose largest logit rises many times along the row.
The bounds are those of finetune_util.py, which know nothing of the shift."""
import pytest

from tests.test_logits_losses_gpu import DTYPES, _stream, check_policy, check_rows, policy_inputs  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# the shifts that leave a type some digits of the logits themselves
SHIFTS = {torch.float32: (30.0, -30.0, 1000.0, -1000.0, 1e5, 5e5), torch.float16: (30.0, -30.0, 1000.0, -3e4),
          torch.bfloat16: (30.0, -100.0, 1000.0, -1e5, 5e5)}


def rising(rows, vocab, shift, dtype, seed):
    """Rows that grow from end to end, in unequal steps; every third row in no order."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g, device="cuda") * 2
    up = x.sort(1).values
    x = torch.where((torch.arange(rows, device="cuda") % 3 != 0)[:, None], up, x)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    t[::2] = vocab - 1 - t[::2] % 7     # likely tokens among them
    return (x + shift).to(dtype), t, g


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
# a row a workgroup, cut rows, odd ends, one vector a wave
@pytest.mark.parametrize("rows,vocab", [(300, 8192), (4, 60001), (270, 50261), (9, 515)])
def test_shifted_rows(rows, vocab, dtype):
    for i, shift in enumerate(SHIFTS[dtype]):
        x, t, g = rising(rows, vocab, shift, dtype, i)
        coef = torch.randn((rows,), generator=g, device="cuda")
        for temperature in (1.0, 0.05):
            check_rows(x, t, coef, temperature, f"shift {shift}")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
# rows held by 256, 512 and 1024 threads, and rows longer than that in float32
@pytest.mark.parametrize("rows,vocab", [(40, 3001), (64, 20011), (30, 60007), (20, 100003)])
def test_policy_of_shifted_rows(rows, vocab, dtype):
    for i, shift in enumerate(SHIFTS[dtype]):
        x, t, g = rising(rows, vocab, shift, dtype, 100 + i)
        for temperature in (1.0, 0.05):
            print(f"case policy shift {shift} {(rows, vocab)} {dtype} T={temperature}", flush=True)
            check_policy(x, t, *policy_inputs(x, t, g, temperature), 0.05, temperature)
