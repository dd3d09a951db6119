"""CPU side of the cache-budget operators: what their entry points refuse
(shapes and types are checked before devices, so no GPU is needed), and the
64-bit oracles against small cases worked out another way."""
import math

import pytest
import torch

from sched_pass_b200 import ops
from sched_pass_b200.models import reference as ref

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def append_args(**kw):
    T, Hq, Hkv, D, P = 3, 4, 2, 64, 5
    a = dict(qkv=torch.zeros(T, (Hq + 2 * Hkv) * D, dtype=BF), q_weight=torch.ones(D, dtype=BF),
             k_weight=torch.ones(D, dtype=BF), eps=1e-5, pos=torch.zeros(T, dtype=I32), slot=torch.zeros(T, dtype=I32),
             cos_sin=torch.zeros(16, D // 2, 2), q_out=torch.zeros(T, Hq, D, dtype=BF),
             k_cache=torch.zeros(P, Hkv, 16, D, dtype=BF), v_cache=torch.zeros(P, Hkv, 16, D, dtype=BF),
             n_q_heads=Hq, n_kv_heads=Hkv, scores=torch.zeros(P, Hkv, 16), positions=torch.zeros(P, Hkv, 16, dtype=I32))
    a.update(kw)
    return a


def scored_args(**kw):
    R, Q, Hq, Hkv, D, P = 2, 1, 4, 2, 64, 5
    a = dict(q=torch.zeros(R, Q, Hq, D, dtype=BF), out=torch.zeros(R, Q, Hq, D, dtype=BF),
             k_cache=torch.zeros(P, Hkv, 16, D, dtype=BF), v_cache=torch.zeros(P, Hkv, 16, D, dtype=BF),
             block_table=torch.zeros(R, 3, dtype=I32), kv_lens=torch.ones(R, dtype=I32), sm_scale=0.125,
             scores=torch.zeros(P, Hkv, 16), lse=torch.zeros(R, Q, Hq), max_len=0)
    a.update(kw)
    return a


def evict_args(**kw):
    R, Hkv, D, P = 2, 2, 64, 5
    a = dict(k_cache=torch.zeros(P, Hkv, 16, D, dtype=BF), v_cache=torch.zeros(P, Hkv, 16, D, dtype=BF),
             scores=torch.zeros(P, Hkv, 16), positions=torch.zeros(P, Hkv, 16, dtype=I32),
             block_table=torch.zeros(R, 3, dtype=I32), kv_lens=torch.ones(R, dtype=I32),
             last_pos=torch.zeros(R, dtype=I32), budget=8, recent=2, sink=1, max_len=0, new_lens=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(qkv=torch.zeros(3, 500, dtype=BF)), "qkv must be"),
    (dict(qkv=torch.zeros(3, 512)), "qkv must have the cache's type"),
    (dict(qkv=torch.zeros(512, 3, dtype=BF).t()), "contiguous rows"),
    (dict(q_weight=torch.ones(32, dtype=BF)), "q_weight and k_weight"),
    (dict(k_weight=torch.ones(64)), "k_weight must have"),
    (dict(pos=torch.zeros(2, dtype=I32)), "pos must be contiguous with at least 3"),
    (dict(slot=torch.zeros(3, dtype=torch.int64)), "slot must be int32"),
    (dict(cos_sin=torch.zeros(16, 12, 2)), "multiple of 16"),
    (dict(cos_sin=torch.zeros(16, 64, 2)), "at most the head dim"),
    (dict(cos_sin=torch.zeros(16, 32, 2, dtype=torch.float64)), "cos_sin must be"),
    (dict(q_out=torch.zeros(2, 4, 64, dtype=BF)), "q_out must be"),
    (dict(n_kv_heads=1), "n_kv_heads must be the cache's"),
    (dict(n_q_heads=0), "n_q_heads must be positive"),
    (dict(v_cache=torch.zeros(4, 2, 16, 64, dtype=BF)), "of one shape"),
    (dict(k_cache=torch.zeros(5, 2, 16, 64)), "bfloat16 or float16"),
    (dict(scores=torch.zeros(5, 2, 15)), "scores must be contiguous"),
    (dict(scores=torch.zeros(5, 2, 16, dtype=BF)), "scores must be float32"),
    (dict(positions=torch.zeros(5, 2, 16)), "positions must be int32"),
    (dict(), "must be a CUDA tensor"),
])
def test_append_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        ops.qk_norm_rope_kv_append(**append_args(**change))


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(2, 1, 3, 64, dtype=BF)), "multiple of the cache's heads"),
    (dict(q=torch.zeros(2, 1, 4, 128, dtype=BF)), "q must be"),
    (dict(q=torch.zeros(2, 1, 4, 64)), "q must have the cache's type"),
    (dict(q=torch.zeros(2, 4, 1, 64, dtype=BF).transpose(1, 2)[..., ::2].repeat(1, 1, 1, 2).transpose(2, 3).contiguous().transpose(2, 3)),
     "contiguous heads"),
    (dict(out=torch.zeros(2, 2, 4, 64, dtype=BF)), "out must have q's shape"),
    (dict(out=torch.zeros(1, 1, 4, 64, dtype=BF).expand(2, 1, 4, 64)), "must not overlap"),
    (dict(block_table=torch.zeros(1, 3, dtype=I32)), "block_table must be"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), "block_table must be int32"),
    (dict(kv_lens=torch.ones(1, dtype=I32)), "kv_lens must be contiguous"),
    (dict(scores=torch.zeros(5, 1, 16)), "scores must be contiguous"),
    (dict(lse=torch.zeros(2, 1, 2)), "lse must be"),
    (dict(lse=torch.zeros(2, 1, 4, dtype=BF)), "lse must be"),
    (dict(max_len=-1), "max_len"),
    (dict(k_cache=torch.zeros(5, 2, 8, 64, dtype=BF), v_cache=torch.zeros(5, 2, 8, 64, dtype=BF)), "multiple of 16"),
    (dict(k_cache=torch.zeros(5, 2, 16, 96, dtype=BF), v_cache=torch.zeros(5, 2, 16, 96, dtype=BF)), "64 or 128"),
    (dict(), "must be a CUDA tensor"),
])
def test_scored_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        ops.attention_decode_scored(**scored_args(**change))


@pytest.mark.parametrize("change,message", [
    (dict(budget=0), "budget must be at least 1"),
    (dict(recent=8, sink=1), "together at most the budget"),
    (dict(recent=-1), "must not be negative"),
    (dict(sink=-1), "must not be negative"),
    (dict(recent=2**31 - 1), "together at most the budget"),
    (dict(max_len=-5), "max_len"),
    (dict(scores=torch.zeros(5, 2, 17)), "scores must be contiguous"),
    (dict(positions=torch.zeros(5, 2, 16)), "positions must be int32"),
    (dict(kv_lens=torch.ones(2, 1, dtype=I32)), "kv_lens must be"),
    (dict(last_pos=torch.zeros(1, dtype=I32)), "last_pos must be contiguous"),
    (dict(new_lens=torch.zeros(1, dtype=I32)), "new_lens must be contiguous"),
    (dict(block_table=torch.zeros(3, 2, dtype=I32).t()), "block_table must be"),
    (dict(v_cache=torch.zeros(5, 2, 16, 64, dtype=torch.float16)), "v_cache must have the cache's type"),
    (dict(), "must be a CUDA tensor"),
])
def test_evict_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        ops.kv_evict(**evict_args(**change))


def test_oracle_append_matches_the_framework_rotation():
    """With unit weights and rows of unit mean square, the norm is the identity
    (eps 0) and the oracle is the framework's rotation."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 3, 64, generator=g, dtype=torch.float64)
    x = x / x.pow(2).mean(-1, keepdim=True).sqrt()
    ang = torch.rand(32, 32, generator=g) * 6
    cs = torch.stack([ang.cos(), ang.sin()], -1)
    pos = torch.tensor([0, 3, 31, 7, 7])
    got = ref.qk_norm_rope(x, torch.ones(64), 0.0, pos, cs)
    want = ref.rope(x, pos, cs)
    assert (got - want).abs().max() < 1e-5  # `rope` rounds to fp32
    part = ref.qk_norm_rope(x, torch.ones(64), 0.0, pos, cs[:, :16])
    assert torch.allclose(part[..., 32:], x[..., 32:], atol=1e-12)


def test_oracle_scored_is_the_decode_oracle_and_its_weights_sum_to_the_rows():
    g = torch.Generator().manual_seed(1)
    P, Hkv, D, Hq = 9, 2, 64, 6
    k, v = (torch.randn(P, Hkv, 16, D, generator=g) for _ in range(2))
    bt = torch.tensor([[4, 2, 0], [1, 8, 3]], dtype=I32)
    lens = torch.tensor([37, 18], dtype=I32)
    q = torch.randn(2, 2, Hq, D, generator=g)
    out, lse, w = ref.attention_scored(q, k, v, bt, lens, 0.125)
    want = ref.decode_attention_paged(q[:, 1], k, v, bt, lens, 0.125)
    assert (out[:, 1] - want).abs().max() < 1e-5
    want0 = ref.decode_attention_paged(q[:, 0], k, v, bt, lens - 1, 0.125)
    assert (out[:, 0] - want0).abs().max() < 1e-5
    for r in range(2):
        assert torch.allclose(w[r].sum(-1), torch.full((Hkv,), 2.0 * Hq / Hkv, dtype=torch.float64))
    bt[0, 1] = 99  # a page outside the cache: its tokens are not there
    out2, _, w2 = ref.attention_scored(q, k, v, bt, lens, 0.125)
    assert w2[0][:, 16:32].abs().max() == 0 and torch.equal(out2[1], out[1])
    empty = ref.attention_scored(q, k, v, bt, torch.tensor([0, 1]), 0.125)
    assert empty[0][0].abs().max() == 0 and empty[1][0].max() == -math.inf and empty[1][1, 0].max() == -math.inf


def test_oracle_evict_by_hand():
    """One head, ten tokens, budget 4: the last two positions and position 0
    stay, then the largest weight; what stays behind the budget fills the holes."""
    k = torch.arange(32.0).view(2, 1, 16, 1).repeat(1, 1, 1, 64)
    v = -k
    scores = torch.zeros(2, 1, 16)
    pos = torch.arange(32, dtype=I32).view(2, 1, 16) - 16  # page 1 holds positions 0..15
    scores[1, 0, :10] = torch.tensor([0., 5, 1, math.nan, 7, 7, 2, math.inf, 0, 0])
    bt, lens, last = torch.tensor([[1, 0]], dtype=I32), torch.tensor([10], dtype=I32), torch.tensor([9], dtype=I32)
    nk, nv, ns, npos, nl = ref.kv_evict(k, v, scores, pos, bt, lens, last, 4, 2, 1)
    # kept: 8, 9 (recent), 0 (sink), 7 (inf); movers 7, 8, 9 into 1, 2, 3
    assert npos[1, 0, :4].tolist() == [0, 7, 8, 9] and nl.tolist() == [4]
    assert nk[1, 0, :4, 0].tolist() == [16, 23, 24, 25] and nv[1, 0, 1, 3] == -23
    assert torch.equal(nk[1, 0, 4:], k[1, 0, 4:]) and torch.equal(nk[0], k[0])
    # equal weights: the lowest slot stays; NaN goes before any number
    nk, _, _, npos, _ = ref.kv_evict(k, v, scores, pos, bt, lens, last, 9, 0, 0)
    assert npos[1, 0, :10].tolist() == [0, 1, 2, 9, 4, 5, 6, 7, 8, 9]
    # a request within its budget is left alone
    same = ref.kv_evict(k, v, scores, pos, bt, lens, last, 10, 2, 0)
    assert torch.equal(same[0], k) and same[4].tolist() == [10]


def test_oracle_evict_leaves_bad_pages_out():
    k = torch.randn(3, 1, 16, 64)
    scores = torch.rand(3, 1, 16) + 1
    scores[0] += 10
    pos = torch.arange(48, dtype=I32).view(3, 1, 16)
    bt = torch.tensor([[0, 7, 2]], dtype=I32)  # slots 16..31 are in no page
    got = ref.kv_evict(k, k, scores, pos, bt, torch.tensor([40]), torch.tensor([100]), 20, 0, 0)
    # 16 tokens of page 0 and 4 of page 2 are kept; the holes are in the bad page: nothing moves
    assert torch.equal(got[0], k) and torch.equal(got[3], pos) and got[4].tolist() == [20]
