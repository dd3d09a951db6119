"""The cache-budget kernels where their arithmetic, scratch and scheduling can
go wrong: weights far below the largest, calls that need scratch on two streams
and in graphs, long runs of tiles, uneven batches.

Tolerances count roundings, as in test_gpu_kv_budget.py.
"""
import pytest
import torch

from sched_pass_b200 import _ext, ops
from sched_pass_b200.models import reference as ref
from test_gpu_kv_budget import BF, DEV, FP, gen, i32, paged

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _clean_status():
    ops.check_status()
    yield
    ops.check_status()


# ------------------------------------------------------------------ weights far below the largest
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("gap", [9.0, 14.0, 17.0, 20.0])
@pytest.mark.parametrize("lens,Q,Hq,Hkv,D,launches", [
    ([8000], 1, 8, 2, 128, 1), ([500] * 16, 1, 16, 8, 128, 1), ([256, 200] * 100, 1, 2, 1, 64, 1),
    ([1600] * 40, 1, 32, 8, 128, 2), ([1600] * 40, 1, 8, 8, 64, 2), ([900, 2000], 5, 16, 2, 128, 2),
    ([120] * 60, 3, 48, 8, 64, 2)])
def test_scored_many_light_tokens_behind_a_heavy_one(lens, Q, Hq, Hkv, D, launches, gap, dtype):
    """The first token of each request outweighs every other by e^gap and has
    the value 0, so the output is the light tokens' alone: their weights must
    keep the type's bits, whatever the largest is."""
    g = gen(int(gap))
    bt, P = paged(lens, 16)
    kc = torch.zeros(P, Hkv, 16, D, dtype=dtype, device=DEV)
    vc = (2e4 * (0.5 + torch.rand(P, Hkv, 16, D, generator=g, device=DEV))).to(dtype)
    first = bt[:, 0].long()
    kc[first, :, 0, 0] = gap
    vc[first, :, 0] = 0
    q = torch.zeros(len(lens), Q, Hq, D, dtype=dtype, device=DEV)
    q[..., 0] = 1
    out, lse, scores = torch.empty_like(q), torch.empty(q.shape[:3], device=DEV), torch.zeros(P, Hkv, 16, device=DEV)
    n0 = _ext.launches()
    ops.attention_decode_scored(q, out, kc, vc, bt, i32(lens), 1.0, scores, lse=lse)
    assert _ext.launches() - n0 == launches
    want, z, _ = ref.attention_scored(q, kc, vc, bt, i32(lens), 1.0)
    u, n = torch.finfo(dtype).eps / 2, max(lens)
    # all terms are positive. The result rounds once (u; a subnormal fp16 one by 2^-25), each weight once (u, all bits
    # kept: 2^-29 < e^-20 of the largest); the logit's scale, its difference to the reference and the exponential are
    # off by 2^-24, 2^-24 of the logit and 2^-22, in both the weight and the sum; n + 64 roundings in each sum.
    tol = (2 * u + u * u + 2 * (gap * 2.0**-22 + 2.0**-22) + 2 * (n + 64) * 2.0**-24) * want + 2.0**-25
    err = (out.double() - want).abs()
    assert bool((err <= tol).all()), (err / tol).max()
    assert bool(((lse.double() - z).abs() <= gap * 2.0**-21 + 2.0**-20 + (n + 8) * 2.0**-24).all())
