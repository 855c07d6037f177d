"""Plans with shared prefixes on the kernels and in the batches beside decode steps on a
16-bit cache: the generic kernel where an MFMA plan shares, prompts over fp8 and 4-bit caches."""
import pytest

from tests.test_gpu_prefix import plan_of, run, share
from tests.window_helpers import BF, F8, F16, F32, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,dtype,kv", [(64, BF, F32), (128, BF, F16), (64, F16, BF), (128, F16, F32)])
@pytest.mark.parametrize("ql", [[1, 1, 1], [1, 30, 3]])
def test_generic_kernel_takes_a_plan_that_shares(D, dtype, kv, ql):
    """A cache dtype that the MFMA kernels do not read, over a plan whose items and
    partials are theirs: every sequence reads its own keys."""
    b = Batch([560, 530, 541], ql, Hq=8, Hkv=2, D=D, dtype=dtype, kv=kv)
    groups = [([0, 1, 2], 528)]
    plan = plan_of(share(b, groups), groups)
    assert plan.info["prefix_items"] > 0
    b.check(run(b, groups, plan), None, 0)


@pytest.mark.parametrize("D,dtype,kv", [(64, BF, F8), (128, BF, "4"), (128, F16, F8), (64, F16, "4"), (128, F16, F16)])
@pytest.mark.parametrize("stride", [0, 80])
def test_prompts_beside_a_group(D, dtype, kv, stride):
    """Two groups, one with a prompt among its members, prompts and a decode row outside them."""
    b = Batch([700, 640, 560, 20, 610, 545, 530, 1500], [1, 3, 70, 80, 2, 1, 1, 1], Hq=8, Hkv=2, D=D, dtype=dtype, kv=kv,
              stride=stride, seed=D)
    groups = [([2, 0, 4], 548), ([6, 5], 520)]
    plan = plan_of(share(b, groups), groups)
    assert plan.info["prefill_seqs"] == 2 and plan.info["prefix_items"] > 0
    b.check(run(b, groups, plan), None, 0)
