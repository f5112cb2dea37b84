"""Fine-tuning operators over more rows than one launch's workgroups or threads."""
import ctypes

import pytest

from tensorplay_amd import _capi
from tests import finetune_util as F
from tests.test_logits_losses_gpu import _stream, check_policy, check_rows, make, policy_inputs  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_rows_past_the_workgroups_of_a_launch():
    """2^24 rows of one workgroup each are cut in two launches, statistics and gradient."""
    rows = (1 << 24) + 70
    x, t, g = make(rows, 5, torch.float16, 50)
    t[-3:] = torch.tensor([-100, 4, 0], device="cuda")
    coef = torch.randn((rows,), generator=g, device="cuda")
    coef[-9] = 0.0
    check_rows(x, t, coef, 1.0, "many rows")


def test_policy_rows_past_the_workgroups_of_a_launch():
    rows = (1 << 24) + 70
    x, t, g = make(rows, 3, torch.bfloat16, 51)
    print(f"case policy {rows}", flush=True)
    old, adv, ref, w = policy_inputs(x, t, g, 1.0)
    w[-5:] = torch.tensor([1.0, 0.0, 2.0, 0.0, 0.5], device="cuda")
    check_policy(x, t, old, adv, ref, w, 0.05, 1.0)


def test_dropout_past_the_threads_of_a_launch():
    """2^32 rows of one column, a thread each: cut a little below 2^32, in place."""
    rows = 1 << 32
    x = torch.ones((rows, 1), dtype=torch.float16, device="cuda")
    p, s = ctypes.c_void_p(x.data_ptr()), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    print(f"case dropout {rows}", flush=True)
    _capi._check(_capi.lib().tpr_dropout(p, _capi.FLOAT16, rows, 1, 0.25, 9, 4, p, s))
    cut = (0xFFFFFFFF // 256) * 256
    for r0 in (0, (1 << 31) - 50, cut - 120, cut - 1, rows - 200):
        n = min(200, rows - r0)
        keep, up = F.keep64(n, 1, 0.25, 9, 4, row0=r0)
        ref = keep.to("cuda") * up
        F.assert_within(x[r0:r0 + n], ref, (2 * F.U + F.HALF[torch.float16]) * ref, f"rows from {r0}")
    del x
    torch.cuda.empty_cache()
