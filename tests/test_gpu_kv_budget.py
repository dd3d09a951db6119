"""The cache-budget kernels (per-head norm + rotation + append, scored decode
attention, eviction) against their 64-bit statements.

Tolerances count roundings. u = half a step of the 16-bit type
(finfo.eps / 2); fp32 operations are off by 2^-24 each, ``ex2.approx`` and
``rsqrtf`` by at most 2^-22 relative.
"""
import math

import pytest
import torch

from sched_pass_b200 import ops
from sched_pass_b200.models import reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _clean_status():
    ops.check_status()
    yield
    ops.check_status()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def expect_bad_index(site, index=None):
    with pytest.raises(ops.KernelStatusError) as e:
        ops.check_status()
    assert (e.value.code, e.value.site) == (7, site) and index in (None, e.value.index), str(e.value)


def paged(lens, page, spare=2, seed=0, cols=None):
    """Shuffled pages for requests of these lengths; unused columns hold -7
    (never to be read). Returns (block table, pages)."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(seed)).tolist()
    bt = torch.full((len(lens), cols or max(max(need), 1)), -7, dtype=torch.int32)
    for r, c in enumerate(need):
        for j in range(c):
            bt[r, j] = order.pop()
    return bt.to(DEV), sum(need) + spare


def rope_table(max_pos, rot):
    ang = torch.arange(max_pos, device=DEV, dtype=torch.float64)[:, None] * (
        10000.0 ** (-torch.arange(rot // 2, device=DEV, dtype=torch.float64) * 2 / rot))
    return torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()


# ------------------------------------------------------------------ norm + rotation + append
def check_append(T, Hq, Hkv, D, rot, dtype, page=16, stride=0, seed=0, track=True, scale=1.0, zero_head=False):
    g = gen(seed)
    width = (Hq + 2 * Hkv) * D
    qkv = (randn(g, T, width + stride) * scale).to(dtype)[:, :width]
    if zero_head and T:
        qkv[0, :D] = 0
    wq, wk = (1 + randn(g, D) * 0.3).to(dtype), (1 + randn(g, D) * 0.3).to(dtype)
    cs = rope_table(300, rot)
    P = T // page + 3
    pos = torch.randint(0, 300, (T,), generator=g, device=DEV).to(torch.int32)
    slot = torch.randperm(P * page, generator=g, device=DEV)[:T].to(torch.int32)
    if T > 2:
        slot[1] = -1
    kc, vc = randn(g, P, Hkv, page, D, dtype=dtype), randn(g, P, Hkv, page, D, dtype=dtype)
    sc, ps = randn(g, P, Hkv, page), torch.full((P, Hkv, page), -3, dtype=torch.int32, device=DEV)
    want = [t.clone() for t in (kc, vc, sc, ps)]
    q_rows = randn(g, T + 1, Hq * D + stride, dtype=dtype)
    last = q_rows.clone()
    q_out = q_rows[:, :Hq * D].view(T + 1, Hq, D) if stride == 0 else q_rows.as_strided((T + 1, Hq, D), (Hq * D + stride, D, 1))
    ops.qk_norm_rope_kv_append(qkv, wq, wk, 1e-5, pos, slot, cs, q_out, kc, vc, Hq, Hkv,
                               scores=sc if track else None, positions=ps if track else None)
    x = qkv.reshape(T, Hq + 2 * Hkv, D)
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps  # a subnormal step

    def near(got, heads, w):
        y = ref.qk_norm_rope(heads, w, 1e-5, pos, cs)
        # each output is a sum of two products: its fp32 error is relative to their magnitudes
        # (norm: D + 8 roundings in the mean, halved by the root; rsqrtf 4, weight 2, rotation 3, spare 3)
        size = ref.qk_norm_rope(heads.double().abs(), w.double().abs(), 1e-5, pos, cs.abs() * torch.tensor([1.0, -1.0], device=DEV))
        size = torch.maximum(size.abs(), ref.qk_norm_rope(heads.double().abs(), w.double().abs(), 1e-5, pos, cs.abs()).abs())
        tol = u * y.abs() + ((D + 8) / 2 + 12) * 2.0**-24 * (1 + u) * size + tiny
        assert bool(((got.double() - y).abs() <= tol).all()), ((got.double() - y).abs() / tol).max()
        return y

    near(q_out[:T], x[:, :Hq], wq)
    on = slot >= 0
    page_i, off = slot[on].long() // page, slot[on].long() % page
    got_k = kc[page_i, :, off]
    full = torch.zeros(T, Hkv, D, dtype=dtype, device=DEV)
    full[on] = got_k
    if bool(on.all()) or T:
        y = ref.qk_norm_rope(x[:, Hq:Hq + Hkv], wk, 1e-5, pos, cs)
        full[~on] = y[~on].to(dtype)
        near(full, x[:, Hq:Hq + Hkv], wk)
    want[0][page_i, :, off] = got_k
    want[1][page_i, :, off] = x[on, Hq + Hkv:]
    if track:
        want[2][page_i, :, off] = 0.0
        want[3][page_i, :, off] = pos[on][:, None].expand(-1, Hkv)
    for t, w in zip((kc, vc, sc, ps), want):
        assert torch.equal(t, w)  # nothing else was written
    assert torch.equal(q_rows[T:], last[T:]) and torch.equal(q_rows[:, Hq * D:], last[:, Hq * D:])


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("T,Hq,Hkv,D,rot", [
    (1, 32, 8, 128, 128), (1, 1, 1, 64, 16), (2, 3, 1, 128, 64), (7, 5, 5, 64, 64), (33, 16, 2, 64, 32),
    (130, 8, 2, 128, 112), (513, 4, 4, 128, 128)])
def test_append_matches(T, Hq, Hkv, D, rot, dtype):
    check_append(T, Hq, Hkv, D, rot, dtype, seed=T)


def test_append_strided_rows_pages_and_untracked():
    check_append(17, 4, 2, 128, 128, BF, page=64, stride=24)
    check_append(5, 4, 2, 64, 64, FP, page=1, stride=8, track=False)
    check_append(40, 6, 3, 64, 32, BF, page=48, track=False)


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 300.0])
def test_append_small_and_large_rows(scale):
    check_append(9, 4, 2, 128, 128, BF, scale=scale, zero_head=True)


@pytest.mark.parametrize("T,Hq,Hkv,D,rot,dtype", [
    (700, 8, 3, 128, 128, BF), (2600, 7, 2, 128, 64, FP), (3100, 5, 1, 64, 64, BF), (9001, 15, 3, 64, 32, FP)])
def test_append_many_tokens(T, Hq, Hkv, D, rot, dtype):
    """The forms for more tokens: several heads to a lane group, with and
    without the pipeline, head counts that do not fill the last group."""
    check_append(T, Hq, Hkv, D, rot, dtype, seed=T)


def test_append_no_tokens():
    check_append(0, 4, 2, 64, 64, BF)


def test_append_infinite_value_stays_in_its_head():
    Hq, Hkv, D = 4, 2, 128
    qkv = randn(gen(1), 2, (Hq + 2 * Hkv) * D, dtype=BF)
    qkv[0, D] = math.inf
    w = torch.ones(D, dtype=BF, device=DEV)
    kc = torch.zeros(2, Hkv, 16, D, dtype=BF, device=DEV)
    vc, q = torch.zeros_like(kc), torch.zeros(2, Hq, D, dtype=BF, device=DEV)
    ops.qk_norm_rope_kv_append(qkv, w, w, 1e-5, i32([0, 1]), i32([0, 1]), rope_table(4, D), q, kc, vc, Hq, Hkv)
    assert bool(torch.isfinite(q[:, [0, 2, 3]]).all()) and bool(torch.isfinite(kc).all())
    assert not bool(torch.isfinite(q[0, 1]).all()) and bool(torch.isfinite(q[1]).all())


def test_append_bad_position_and_slot():
    Hq, Hkv, D = 2, 2, 64
    g = gen(3)
    qkv = randn(g, 3, (Hq + 2 * Hkv) * D, dtype=BF)
    w, cs = torch.ones(D, dtype=BF, device=DEV), rope_table(10, D)
    kc = randn(g, 2, Hkv, 16, D, dtype=BF)
    vc, k0 = kc.clone(), kc.clone()
    q = torch.ones(3, Hq, D, dtype=BF, device=DEV)
    for bad in (10, -1):
        ops.qk_norm_rope_kv_append(qkv, w, w, 1e-5, i32([bad, 3, 4]), i32([5, -1, -1]), cs, q, kc, vc, Hq, Hkv)
        expect_bad_index(7, bad)
        assert q[0].abs().max() == 0 and q[1].abs().max() > 0 and torch.equal(kc, k0) and torch.equal(vc, k0)
    ops.qk_norm_rope_kv_append(qkv, w, w, 1e-5, i32([1, 3, 4]), i32([32, -1, -1]), cs, q, kc, vc, Hq, Hkv)
    expect_bad_index(3, 32)
    assert torch.equal(kc, k0) and torch.equal(vc, k0) and q[0].abs().max() > 0


# ------------------------------------------------------------------ scored attention
def scored_inputs(lens, Q, Hq, Hkv, D, dtype, page=16, seed=0, cols=None, q_scale=1.0):
    g = gen(seed)
    bt, P = paged(lens, page, seed=seed, cols=cols)
    kc, vc = randn(g, P, Hkv, page, D, dtype=dtype), randn(g, P, Hkv, page, D, dtype=dtype)
    q = (randn(g, len(lens), Q, Hq, D) * q_scale).to(dtype)
    scores = torch.rand(P, Hkv, page, generator=g, device=DEV)
    return q, kc, vc, bt, i32(lens), scores


def check_scored(q, kc, vc, bt, lens, scores0, out, lse, scores, scale, bad=()):
    """``bad``: requests not compared (their table was out of range)."""
    R, Q, Hq, D = q.shape
    P, Hkv, ps, _ = kc.shape
    u = torch.finfo(q.dtype).eps / 2
    want, z, weights = ref.attention_scored(q, kc, vc, bt, lens, scale)
    left = scores0.double().clone()
    used = torch.zeros(P, Hkv, ps, dtype=torch.bool, device=DEV)
    for r in range(R):
        n = int(lens[r])
        if r in bad:
            continue
        pages = bt[r, :(n + ps - 1) // ps].long()
        k = kc[pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :n].double() if n else None
        v = vc[pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :n].double() if n else None
        # a logit is a sum of D products in fp32 (D + 4 roundings), its exponential off by 2^-22 more and by the
        # rounding of the logit itself
        most = 0.0 if not n else float((q[r].double().abs().view(Q, Hkv, -1, D).transpose(0, 1).reshape(Hkv, -1, D)
                                        @ torch.nan_to_num(k).abs().transpose(1, 2)).max()) * scale
        delta = (D + 8) * 2.0**-24 * most + 2.0**-20
        for i in range(Q):
            see = max(0, n - (Q - 1 - i))
            if see == 0:
                assert out[r, i].abs().max() == 0
                assert lse is None or bool((lse[r, i] == -math.inf).all())
                continue
            s = torch.einsum("hgd,hnd->hgn", q[r, i].double().view(Hkv, -1, D), k[:, :see]) * scale
            p = torch.softmax(s, -1)
            size = torch.einsum("hgn,hnd->hgd", p, v[:, :see].abs()).reshape(Hq, D)
            # P rounds to the 16-bit type (u; below its normal range by a subnormal step), the sums to fp32,
            # the result to the 16-bit type
            tiny = torch.finfo(q.dtype).tiny * 2 * u
            tol = u * want[r, i].abs() * (1 + u) + (u + 2 * delta + (see + 64) * 2.0**-24) * size + \
                tiny * (1 + v[:, :see].abs().sum(1).repeat_interleave(Hq // Hkv, 0))
            err = (out[r, i].double() - want[r, i]).abs()
            assert bool((err <= tol).all()), (r, i, (err / tol).max())
            if lse is not None:
                e = (lse[r, i].double() - z[r, i]).abs()
                assert bool((e <= delta + (see + 8) * 2.0**-24 + 2.0**-22 * z[r, i].abs()).all()), (r, i, e.max())
        if n:
            w = weights[r]
            padded = torch.zeros(Hkv, pages.numel() * ps, dtype=torch.float64, device=DEV)
            padded[:, :n] = w
            left[pages] += padded.view(Hkv, -1, ps).transpose(0, 1)
            used[pages] = (torch.arange(pages.numel() * ps, device=DEV) < n).view(-1, 1, ps).expand(-1, Hkv, ps)
            rows = Q * Hq // Hkv
            tol = (2 * delta + (rows + 8) * 2.0**-23 + (n + 8) * 2.0**-24) * left[pages] + 2.0**-120
            err = (scores[pages].double() - left[pages]).abs()
            assert bool((err <= tol).all()), (r, (err / tol).max())
    if not bad:
        assert torch.equal(scores[~used], scores0[~used])  # entries behind the ends, and of no request


def run_scored(lens, Q, Hq, Hkv, D, dtype, page=16, seed=0, max_len=0, cols=None, q_scale=1.0):
    q, kc, vc, bt, kl, scores0 = scored_inputs(lens, Q, Hq, Hkv, D, dtype, page, seed, cols, q_scale)
    scores, out = scores0.clone(), torch.full_like(q, 7.0)
    lse = torch.full(q.shape[:3], 7.0, device=DEV)
    r = ops.attention_decode_scored(q, out, kc, vc, bt, kl, D**-0.5, scores, lse=lse, max_len=max_len)
    assert r is out
    check_scored(q, kc, vc, bt, kl, scores0, out, lse, scores, D**-0.5)


LENS = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 300]


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 64), (8, 2, 128), (8, 1, 128), (12, 4, 64), (16, 1, 128), (20, 1, 64)])
def test_scored_lengths_and_groups(Hq, Hkv, D, dtype):
    run_scored(LENS, 1, Hq, Hkv, D, dtype, seed=Hq)


@pytest.mark.parametrize("Q", [2, 3, 16, 40])
@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 128), (8, 2, 64), (6, 2, 128)])
def test_scored_windows(Q, Hq, Hkv, D):
    run_scored([0, 1, 2, 3, 15, 17, 33, 64, 200], Q, Hq, Hkv, D, BF, seed=Q)


def test_scored_most_query_rows():
    """8192 query rows on one KV head, the most a call takes; one more is refused."""
    run_scored([600, 37], 512, 16, 1, 64, BF)
    q, kc, vc, bt, kl, scores = scored_inputs([40], 513, 16, 1, 64, BF)
    with pytest.raises(RuntimeError, match="8192 query rows"):
        ops.attention_decode_scored(q, torch.empty_like(q), kc, vc, bt, kl, 0.125, scores)


def test_scored_thousands_of_requests():
    lens = [0] * 3000
    lens[5], lens[1500], lens[2999], lens[31], lens[32] = 300, 17, 1, 64, 400
    run_scored(lens, 1, 4, 1, 64, BF)


@pytest.mark.parametrize("n,max_len", [(700, 0), (1500, 1500), (2049, 4096), (5001, 5001)])
def test_scored_long(n, max_len):
    run_scored([n, 1, n - 1, n // 2], 1, 8, 2, 128, BF, seed=n, max_len=max_len, cols=-(-max(n, max_len) // 16))


def test_scored_many_requests():
    """Enough (request, head) pairs to fill the device without splitting."""
    run_scored([37 + 13 * (i % 11) for i in range(200)], 1, 8, 8, 64, BF)


@pytest.mark.parametrize("n,Hq,Hkv,D", [(8192, 8, 2, 128), (8100, 16, 1, 64), (4097, 16, 1, 128), (1025, 3, 1, 64)])
def test_scored_one_kernel_form(n, Hq, Hkv, D):
    """Few heads: one kernel, up to its longest contexts, and the two-kernel
    form of the same call among many more requests."""
    from sched_pass_b200 import _ext
    lens = [n, 1, 0, n // 3]
    n0 = _ext.launches()
    run_scored(lens, 1, Hq, Hkv, D, BF, seed=n)
    assert _ext.launches() - n0 == 1
    q, kc, vc, bt, kl, scores0 = scored_inputs(lens, 1, Hq, Hkv, D, BF, seed=n)
    one, s1 = torch.empty_like(q), scores0.clone()
    ops.attention_decode_scored(q, one, kc, vc, bt, kl, D**-0.5, s1)
    many = 40
    q2 = torch.cat([q, torch.zeros(many, 1, Hq, D, dtype=BF, device=DEV)])
    bt2 = torch.cat([bt, torch.zeros(many, bt.shape[1], dtype=torch.int32, device=DEV)])
    two, s2 = torch.empty_like(q2), scores0.clone()
    n0 = _ext.launches()
    ops.attention_decode_scored(q2, two, kc, vc, bt2, torch.cat([kl, torch.zeros(many, dtype=torch.int32, device=DEV)]),
                                D**-0.5, s2)
    assert _ext.launches() - n0 == 2
    assert two[4:].abs().max() == 0
    # sums in another order: a step of the 16-bit result, 2^-18 of the weights
    assert bool(((one.float() - two[:4].float()).abs() <= 2.0**-7 * one.float().abs() + 2.0**-10).all())
    assert bool(((s1 - s2).abs() <= 2.0**-18 * s1).all())


@pytest.mark.parametrize("R,n", [(2, 250), (9, 1000), (16, 500), (30, 500), (64, 250), (130, 100)])
@pytest.mark.parametrize("Hq,D", [(32, 128), (128, 128), (24, 64)])
def test_scored_one_kernel_with_fewer_ctas(R, n, Hq, D):
    """Four, two and one CTA per head, and several waves of one."""
    run_scored([n - (37 * i) % n for i in range(R)], 1, Hq, 8, D, BF, seed=R)


IDLE = [0] * 300  # requests without tokens: with them a call has too many heads for the one-kernel forms


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("Q,Hq,Hkv,D", [(1, 4, 4, 64), (1, 8, 2, 128), (1, 16, 2, 128), (1, 32, 2, 64), (2, 6, 2, 128),
                                        (3, 10, 2, 64), (20, 8, 2, 128)])
def test_scored_two_kernel_form(Q, Hq, Hkv, D, dtype):
    from sched_pass_b200 import _ext
    n0 = _ext.launches()
    run_scored([0, 1, 15, 16, 17, 300, 301, 513, 700, 1023, 64] + IDLE, Q, Hq, Hkv, D, dtype, seed=Hq)
    assert _ext.launches() - n0 == 2


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("Q", [1, 4])
def test_scored_two_kernels_stale_values_and_bad_pages(value, Q):
    lens, Hq, Hkv, D = [289, 7, 300, 641] + IDLE, 8, 2, 128
    q, kc, vc, bt, kl, scores0 = scored_inputs(lens, Q, Hq, Hkv, D, BF)
    clean = (kc.clone(), vc.clone())
    for r, n in enumerate(lens[:4]):
        if n % 16:
            kc[bt[r, n // 16], :, n % 16:] = value
            vc[bt[r, n // 16], :, n % 16:] = value
    scores, out, lse = scores0.clone(), torch.empty_like(q), torch.empty(q.shape[:3], device=DEV)
    ops.attention_decode_scored(q, out, kc, vc, bt, kl, D**-0.5, scores, lse=lse)
    check_scored(q, *clean, bt, kl, scores0, out, lse, scores, D**-0.5)
    table = bt.clone()
    table[2, 3], table[3, 40] = kc.shape[0], -9
    scores = scores0.clone()
    ops.attention_decode_scored(q, out, kc, vc, table, kl, D**-0.5, scores, lse=lse)
    expect_bad_index(8)
    check_scored(q, *clean, bt, kl, scores0, out, lse, scores, D**-0.5, bad=(2, 3))
    want, z, _ = ref.attention_scored(q[:4], *clean, table, kl, D**-0.5)
    assert (out[:4].double() - want).abs().max() < 0.02
    assert (lse[2:4].double() - z[2:4]).abs().max() < 1e-4


@pytest.mark.parametrize("page", [32, 48, 128])
def test_scored_page_sizes(page):
    run_scored([0, 1, 47, 48, 49, 130, 400], 1, 8, 2, 128, BF, page=page)


def test_scored_sharp_softmax():
    """Logits of +-100: one token takes all the weight in most rows."""
    run_scored([5, 90, 333], 1, 8, 2, 128, BF, q_scale=12.0)


def test_scored_single_query_form_and_strides():
    """q [R, Hq, D] as a view of the fused projection's rows, out likewise."""
    Hq, Hkv, D, lens = 8, 2, 128, [33, 0, 64]
    q, kc, vc, bt, kl, scores0 = scored_inputs(lens, 1, Hq, Hkv, D, BF)
    rows = randn(gen(9), 3, (Hq + 2 * Hkv) * D, dtype=BF)
    rows[:, :Hq * D] = q.view(3, -1)
    q3 = rows[:, :Hq * D].view(3, Hq, D)
    ob = torch.full((3, Hq * D + 40), 5.0, dtype=BF, device=DEV)
    out = ob[:, :Hq * D].view(3, Hq, D)
    table = torch.full((5, bt.shape[1] + 3), 10**6, dtype=torch.int32, device=DEV)
    table[:3, :bt.shape[1]] = bt
    scores, lse = scores0.clone(), torch.empty(3, Hq, device=DEV)
    ops.attention_decode_scored(q3, out, kc, vc, table, kl, D**-0.5, scores, lse=lse, max_len=64)
    check_scored(q, kc, vc, bt, kl, scores0, out.unsqueeze(1), lse.unsqueeze(1), scores, D**-0.5)
    assert bool((ob[:, Hq * D:] == 5.0).all())
    again = ops.attention_decode_scored(q3, torch.empty_like(q3.contiguous()), kc, vc, table, kl, D**-0.5, scores0.clone())
    assert torch.equal(again, out)  # without lse, over the whole table width


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("Q", [1, 4])
def test_scored_stale_values_behind_the_end(value, Q):
    """What a page holds behind a request's end takes no part, whatever it is."""
    lens, Hq, Hkv, D = [1, 7, 16, 41], 8, 2, 128
    q, kc, vc, bt, kl, scores0 = scored_inputs(lens, Q, Hq, Hkv, D, BF)
    clean = (kc.clone(), vc.clone())
    for r, n in enumerate(lens):
        if n % 16:
            kc[bt[r, n // 16], :, n % 16:] = value
            vc[bt[r, n // 16], :, n % 16:] = value
    scores, out, lse = scores0.clone(), torch.empty_like(q), torch.empty(q.shape[:3], device=DEV)
    ops.attention_decode_scored(q, out, kc, vc, bt, kl, D**-0.5, scores, lse=lse)
    check_scored(q, *clean, bt, kl, scores0, out, lse, scores, D**-0.5)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("Hq", [2, 8])
def test_scored_nan_in_the_newest_tokens_stays_with_the_queries_that_see_them(which, Hq):
    lens, Q, Hkv, D = [40], 4, 2, 128
    q, kc, vc, bt, kl, scores0 = scored_inputs(lens, Q, Hq, Hkv, D, BF)
    clean = (kc.clone(), vc.clone())
    (kc if which == "k" else vc)[bt[0, 38 // 16], :, 38 % 16] = math.nan  # seen by the last two of the four queries
    scores, out, lse = scores0.clone(), torch.empty_like(q), torch.empty(q.shape[:3], device=DEV)
    ops.attention_decode_scored(q, out, kc, vc, bt, kl, D**-0.5, scores, lse=lse)
    want, z, _ = ref.attention_scored(q, *clean, bt, kl, D**-0.5)
    assert bool(torch.isnan(out[0, 2:]).all())
    assert (out[0, :2].double() - want[0, :2]).abs().max() < 0.02
    assert (lse[0, :2].double() - z[0, :2]).abs().max() < 1e-4
    assert bool(torch.isnan(lse[0, 2:]).all()) == (which == "k")


def test_scored_all_logits_nan():
    q, kc, vc, bt, kl, scores0 = scored_inputs([20, 20], 1, 4, 2, 64, BF)
    kc[bt[0].long()] = math.nan
    scores, out = scores0.clone(), torch.empty_like(q)
    ops.attention_decode_scored(q, out, kc, vc, bt, kl, 0.125, scores)
    assert bool(torch.isnan(out[0]).all()) and bool(torch.isfinite(out[1]).all())


def test_scored_bad_pages_and_lengths():
    lens, Hq, Hkv, D = [50, 40, 64], 4, 2, 64
    q, kc, vc, bt, kl, scores0 = scored_inputs(lens, 1, Hq, Hkv, D, BF)
    P = kc.shape[0]
    for bad in (P, -1, 2**31 - 1):
        table = bt.clone()
        table[1, 1] = bad
        scores, out, lse = scores0.clone(), torch.empty_like(q), torch.empty(q.shape[:3], device=DEV)
        ops.attention_decode_scored(q, out, kc, vc, table, kl, D**-0.5, scores, lse=lse)
        expect_bad_index(8, bad)
        check_scored(q, kc, vc, bt, kl, scores0, out, lse, scores, D**-0.5, bad=(1,))
        want, z, w = ref.attention_scored(q, kc, vc, table, kl, D**-0.5)
        assert (out[1].double() - want[1]).abs().max() < 0.02 and (lse[1].double() - z[1]).abs().max() < 1e-4
    # all of a request's pages bad: an empty row
    table = bt.clone()
    table[0] = -1
    scores, out = scores0.clone(), torch.empty_like(q)
    ops.attention_decode_scored(q, out, kc, vc, table, kl, D**-0.5, scores)
    expect_bad_index(8, -1)
    assert out[0].abs().max() == 0
    # a length behind the table's end or the caller's bound is cut; a negative one is empty
    scores, out = scores0.clone(), torch.empty_like(q)
    ops.attention_decode_scored(q, out, kc, vc, bt, i32([50, -4, 1000]), D**-0.5, scores)
    expect_bad_index(9, 1000)
    check_scored(q, kc, vc, bt, i32([50, 0, 64]), scores0, out, None, scores, D**-0.5)
    scores, out = scores0.clone(), torch.empty_like(q)
    ops.attention_decode_scored(q, out, kc, vc, bt, kl, D**-0.5, scores, max_len=45)
    expect_bad_index(9)
    check_scored(q, kc, vc, bt, i32([45, 40, 45]), scores0, out, None, scores, D**-0.5)


def test_scored_shared_pages_add_up():
    """Two requests on the same pages: each adds its weights."""
    q, kc, vc, bt, kl, scores0 = scored_inputs([40, 40], 1, 4, 2, 64, BF)
    bt[1] = bt[0]
    scores, out = scores0.clone(), torch.empty_like(q)
    ops.attention_decode_scored(q, out, kc, vc, bt, kl, 0.125, scores)
    _, _, w = ref.attention_scored(q, kc, vc, bt, kl, 0.125)
    got = (scores.double() - scores0.double())[bt[0].long()].transpose(0, 1).reshape(2, -1)[:, :40]
    assert (got - (w[0] + w[1])).abs().max() < 1e-5


def test_scored_repeats_bit_for_bit():
    q, kc, vc, bt, kl, scores0 = scored_inputs([900, 333], 1, 8, 2, 128, BF)
    res = []
    for _ in range(3):
        scores, out = scores0.clone(), torch.empty_like(q)
        ops.attention_decode_scored(q, out, kc, vc, bt, kl, 0.09, scores)
        res.append((out, scores))
    assert all(torch.equal(a, b) for x in res[1:] for a, b in zip(x, res[0]))


# ------------------------------------------------------------------ eviction
def evict_inputs(lens, Hkv, D, dtype, page=16, seed=0, kind="lognormal", cols=None):
    g = gen(seed)
    bt, P = paged(lens, page, seed=seed, cols=cols)
    kc, vc = randn(g, P, Hkv, page, D, dtype=dtype), randn(g, P, Hkv, page, D, dtype=dtype)
    shape = (P, Hkv, page)
    scores = torch.exp(2 * randn(g, *shape))
    if kind == "equal":
        scores = torch.full(shape, 0.25, device=DEV)
    elif kind == "ties":
        scores = torch.randint(0, 4, shape, generator=g, device=DEV).float()
    elif kind == "zeros":
        scores = torch.where(torch.rand(shape, generator=g, device=DEV) < 0.5, 0.0, -0.0)
    elif kind == "odd":
        pick = torch.randint(0, 8, shape, generator=g, device=DEV)
        for i, x in enumerate((math.nan, math.inf, -math.inf, -1.5, 1e-42, 3e38)):
            scores[pick == i] = x
    pos = torch.full(shape, -1, dtype=torch.int32, device=DEV)
    last = []
    for r, n in enumerate(lens):
        pages = bt[r, :-(-n // page)].long()
        for h in range(Hkv):
            p = torch.randperm(2 * n + 1, generator=g, device=DEV)[:pages.numel() * page]
            row = torch.full((pages.numel() * page,), -1, dtype=torch.int32, device=DEV)
            row[:p.numel()] = p.to(torch.int32)
            pos[pages, h] = row.view(-1, page)
        last.append(2 * n)
    return kc, vc, scores, pos, bt, i32(lens), i32(last)


def check_evict(state, budget, recent, sink, max_len=0):
    want = ref.kv_evict(*state, budget, recent, sink)
    got = [t.clone() for t in state[:4]]
    lens0 = state[5].clone()
    lens = ops.kv_evict(*got, *state[4:], budget, recent, sink=sink, max_len=max_len)
    for name, a, b in zip(("k", "v", "scores", "positions"), got, want):
        assert torch.equal(torch.nan_to_num(a.float(), nan=-77.0), torch.nan_to_num(b.float(), nan=-77.0)), name
    assert lens.dtype == torch.int32 and torch.equal(lens, want[4]) and torch.equal(state[5], lens0)


@pytest.mark.parametrize("kind", ["lognormal", "equal", "ties", "zeros", "odd"])
@pytest.mark.parametrize("budget,recent,sink", [(1, 0, 0), (1, 1, 0), (16, 4, 2), (64, 64, 0), (100, 30, 4), (299, 0, 299)])
def test_evict_matches(kind, budget, recent, sink):
    check_evict(evict_inputs([0, 1, 2, 16, 17, 65, 100, 101, 300], 3, 64, BF, kind=kind), budget, recent, sink)


@pytest.mark.parametrize("D,dtype,page", [(128, BF, 16), (128, FP, 32), (64, FP, 7), (128, BF, 1)])
def test_evict_layouts(D, dtype, page):
    check_evict(evict_inputs([250, 64, 33], 2, D, dtype, page=page, seed=page), 33, 8, 1)


@pytest.mark.parametrize("n,budget", [(1024, 1023), (1025, 1000), (4000, 1000), (9000, 8000), (41000, 20000), (45001, 77)])
def test_evict_long(n, budget):
    """Up to contexts whose keys do not fit shared memory."""
    check_evict(evict_inputs([n, n // 2], 1, 64, BF, seed=n), budget, budget // 4, 4)


def test_evict_many_heads_and_moves():
    """A CTA per head, with more moves than it lists at a time."""
    check_evict(evict_inputs([5000 - 7 * i for i in range(19)], 8, 64, BF, seed=3), 2400, 100, 4)


def test_evict_unaligned_tracking_tensors():
    """scores and positions that do not start on a 16-byte boundary take the scalar loads."""
    state = evict_inputs([300, 150], 2, 64, BF)
    want = ref.kv_evict(*state, 100, 10, 2)
    got = [t.clone() for t in state[:4]]
    for i in (2, 3):
        room = torch.empty(got[i].numel() + 1, dtype=got[i].dtype, device=DEV)
        got[i] = room[1:].view(got[i].shape).copy_(state[i])
    lens = ops.kv_evict(*got, *state[4:], 100, 10, sink=2)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(lens, want[4])


def test_evict_more_protected_than_the_budget():
    """Positions that repeat protect more tokens than fit: the lowest slots stay."""
    state = evict_inputs([90], 2, 64, BF)
    state[3].fill_(0)
    state[3][state[4][0, 0].long()] = 5
    check_evict(state, 30, 0, 1)


def test_evict_bounds_of_the_host():
    """The table is wider than any request; a bound below the budget moves nothing."""
    state = evict_inputs([50, 20], 2, 64, BF, cols=40)
    check_evict(state, 30, 5, 0, max_len=50)
    check_evict(state, 50, 5, 0, max_len=50)
    check_evict(state, 5000, 5, 0)


def test_evict_bad_pages_and_lengths():
    state = list(evict_inputs([80, 70], 2, 64, BF))
    P = state[0].shape[0]
    for col, bad in ((0, P), (4, -1), (2, 2**31 - 1)):
        broken = list(state)
        broken[4] = state[4].clone()
        broken[4][0, col] = bad
        want = ref.kv_evict(*broken, 40, 6, 2)
        got = [t.clone() for t in state[:4]]
        lens = ops.kv_evict(*got, *broken[4:], 40, 6, sink=2)
        expect_bad_index(10, bad)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(lens, want[4])
    cut = list(state)
    cut[5] = i32([80, 500])  # the table holds 80
    got = [t.clone() for t in state[:4]]
    lens = ops.kv_evict(*got, state[4], cut[5], state[6], 100, 6)
    expect_bad_index(11, 500)
    assert lens.tolist() == [80, 80] and all(torch.equal(a, b) for a, b in zip(got, state[:4]))
    got = [t.clone() for t in state[:4]]
    lens = ops.kv_evict(*got, state[4], i32([-3, 0]), state[6], 10, 6)
    assert lens.tolist() == [0, 0] and all(torch.equal(a, b) for a, b in zip(got, state[:4]))


def test_evict_refuses_its_lengths_as_output():
    state = evict_inputs([50, 20], 2, 64, BF)
    with pytest.raises(RuntimeError, match="must not overlap"):
        ops.kv_evict(*state, 30, 5, new_lens=state[5])


# ------------------------------------------------------------------ as they are used
class Budget:
    """A small decode loop over one layer: append, attend, evict."""

    def __init__(self, R=3, Hq=8, Hkv=2, D=128, budget=40, slack=8, dtype=BF, seed=0):
        g = gen(seed)
        self.R, self.Hq, self.Hkv, self.D, self.budget, self.slack = R, Hq, Hkv, D, budget, slack
        cols = -(-(budget + slack) // 16)
        self.bt = torch.randperm(R * cols, generator=g, device=DEV).to(torch.int32).view(R, cols)
        P = R * cols
        self.kc, self.vc = (torch.zeros(P, Hkv, 16, D, dtype=dtype, device=DEV) for _ in range(2))
        self.scores = torch.zeros(P, Hkv, 16, device=DEV)
        self.positions = torch.zeros(P, Hkv, 16, dtype=torch.int32, device=DEV)
        self.wq, self.wk = (1 + 0.2 * randn(g, D)).to(dtype), (1 + 0.2 * randn(g, D)).to(dtype)
        self.cs = rope_table(512, D)
        self.lens = torch.zeros(R, dtype=torch.int32, device=DEV)
        self.pos = torch.zeros(R, dtype=torch.int32, device=DEV)
        self.qkv = torch.zeros(R, (Hq + 2 * Hkv) * D, dtype=dtype, device=DEV)
        self.q = torch.empty(R, Hq, D, dtype=dtype, device=DEV)
        self.out = torch.empty_like(self.q)

    def state(self):
        return [self.kc, self.vc, self.scores, self.positions]

    def step(self):
        """One token of every request, then back to the budget (lengths stay on the device)."""
        r = torch.arange(self.R, device=DEV)
        slot = self.bt[r, (self.lens // 16).long()] * 16 + self.lens % 16
        ops.qk_norm_rope_kv_append(self.qkv, self.wq, self.wk, 1e-5, self.pos, slot, self.cs, self.q, self.kc, self.vc,
                                   self.Hq, self.Hkv, scores=self.scores, positions=self.positions)
        lens = self.lens + 1
        ops.attention_decode_scored(self.q, self.out, self.kc, self.vc, self.bt, lens, self.D**-0.5, self.scores,
                                    max_len=self.budget + self.slack)
        cut = ops.kv_evict(self.kc, self.vc, self.scores, self.positions, self.bt, lens, self.pos, self.budget, 8,
                           sink=2, max_len=self.budget + self.slack)
        self.lens.copy_(cut)
        self.pos += 1


def test_decode_under_a_budget():
    """Sixty steps: each step's kernels against the oracles on the state they
    started from, so that errors cannot add up unseen; lengths stay at the budget."""
    b = Budget()
    g = gen(11)
    for step in range(60):
        b.qkv.copy_(randn(g, *b.qkv.shape))
        before = [t.clone() for t in b.state()]
        lens, pos = b.lens.clone(), b.pos.clone()
        b.step()
        x = b.qkv.view(b.R, -1, b.D)
        kc, vc, sc, ps = before
        for r in range(b.R):
            page, off = int(b.bt[r, int(lens[r]) // 16]), int(lens[r]) % 16
            kc[page, :, off] = ref.qk_norm_rope(x[r:r + 1, b.Hq:b.Hq + b.Hkv], b.wk, 1e-5, pos[r:r + 1], b.cs)[0].to(BF)
            vc[page, :, off] = x[r, b.Hq + b.Hkv:]
            sc[page, :, off] = 0
            ps[page, :, off] = pos[r]
        q = ref.qk_norm_rope(x[:, :b.Hq], b.wq, 1e-5, pos, b.cs).to(BF)
        n = lens + 1
        out, _, w = ref.attention_scored(q[:, None], kc, vc, b.bt, n, b.D**-0.5)
        assert (b.out.double() - out[:, 0]).abs().max() < 0.03
        for r in range(b.R):
            pages = b.bt[r].long()
            add = torch.zeros(b.Hkv, pages.numel() * 16, dtype=torch.float64, device=DEV)
            add[:, :int(n[r])] = w[r]
            sc[pages] += add.view(b.Hkv, -1, 16).transpose(0, 1).float()
        want = ref.kv_evict(kc, vc, sc, ps, b.bt, n, pos, b.budget, 8, 2)
        assert torch.equal(b.lens, want[4])
        for r in range(b.R):
            for h in range(b.Hkv):
                m = int(b.lens[r])
                got_p = b.positions[b.bt[r].long(), h].reshape(-1)[:m]
                want_p = want[3][b.bt[r].long(), h].reshape(-1)[:m]
                # weights agree to fp32 rounding: the kept sets may differ only where two weights nearly tie
                same = torch.isin(got_p, want_p).sum()
                assert int(same) >= m - 1 and got_p.unique().numel() == m
                assert int((got_p > pos[r] - 8).sum()) == min(8, m) and {0, 1} & set(got_p.tolist()) == {0, 1} & set(range(int(pos[r]) + 1))


def test_captured_steps_equal_eager_ones():
    """The three operators in one graph, replayed with new inputs, beside an
    eager copy; and two graphs replayed alternately."""
    eager, a, c = Budget(seed=5), Budget(seed=5), Budget(seed=6)
    other = Budget(seed=6)
    graphs = []
    side = torch.cuda.Stream()
    for x in (a, c):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            snap = [t.clone() for t in (*x.state(), x.lens, x.pos)]
            x.step()
            for t, s in zip((*x.state(), x.lens, x.pos), snap):
                t.copy_(s)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            x.step()
        graphs.append(gr)
    g = gen(3)
    for _ in range(52):
        rows = randn(g, *a.qkv.shape)
        for x in (eager, a, c, other):
            x.qkv.copy_(rows)
        eager.step()
        graphs[0].replay()
        graphs[1].replay()
        other.step()
    for x, y in ((eager, a), (other, c)):
        assert torch.equal(x.out, y.out) and torch.equal(x.lens, y.lens) and torch.equal(x.pos, y.pos)
        assert all(torch.equal(s, t) for s, t in zip(x.state(), y.state()))


def test_two_streams_at_once():
    """Independent states stepped on two streams: no scratch is shared."""
    pair, alone = [Budget(seed=s, R=16, budget=200, slack=24) for s in (1, 2)], [Budget(seed=s, R=16, budget=200, slack=24) for s in (1, 2)]
    rows = randn(gen(4), 30, *pair[0].qkv.shape, dtype=BF)
    streams = [torch.cuda.Stream() for _ in pair]
    torch.cuda.synchronize()
    for i in range(30):
        for x, st in zip(pair, streams):
            with torch.cuda.stream(st):
                x.qkv.copy_(rows[i])
                x.step()
    torch.cuda.synchronize()
    for i in range(30):
        for x in alone:
            x.qkv.copy_(rows[i])
            x.step()
    for x, y in zip(pair, alone):
        assert torch.equal(x.out, y.out) and all(torch.equal(s, t) for s, t in zip(x.state(), y.state()))


def test_long_cache_offsets_pass_32_bits():
    """Pages whose element offsets lie beyond 2^32 (a cache of 4.4e9 elements)."""
    P, Hkv, ps, D = 270000, 8, 16, 128
    kc = torch.empty(P, Hkv, ps, D, dtype=BF, device=DEV)
    vc = torch.empty_like(kc)
    scores = torch.zeros(P, Hkv, ps, device=DEV)
    positions = torch.zeros(P, Hkv, ps, dtype=torch.int32, device=DEV)
    g = gen(2)
    last = torch.tensor([P - 1, P - 3, P - 2, 5], device=DEV)
    kc[last], vc[last] = randn(g, 4, Hkv, ps, D, dtype=BF), randn(g, 4, Hkv, ps, D, dtype=BF)
    bt = last.to(torch.int32).view(1, 4)
    q = randn(g, 1, 1, 16, D, dtype=BF)
    out, lens = torch.empty_like(q), i32([60])
    qkv = randn(g, 1, 32 * D, dtype=BF)
    w = torch.ones(D, dtype=BF, device=DEV)
    ops.qk_norm_rope_kv_append(qkv, w, w, 1e-5, i32([59]), i32([5 * 16 + 11]), rope_table(64, D), q[:, 0], kc, vc, 16, Hkv,
                               scores=scores, positions=positions)
    ops.attention_decode_scored(q, out, kc, vc, bt, lens, D**-0.5, scores)
    small = (kc[last].clone(), vc[last].clone())
    order = i32([[0, 1, 2, 3]])
    check_scored(q, *small, order, lens, torch.zeros(4, Hkv, ps, device=DEV), out, None, scores[last], D**-0.5)
    positions[last] = torch.arange(64, device=DEV).to(torch.int32).view(4, 1, 16).expand(4, Hkv, 16)
    want = ref.kv_evict(*small, scores[last].clone(), positions[last].clone(), order, lens, i32([59]), 20, 4, 2)
    ops.kv_evict(kc, vc, scores, positions, bt, lens, i32([59]), 20, 4, sink=2)
    for a, b in zip((kc, vc, scores, positions), want):
        assert torch.equal(a[last], b)


def test_scratch_that_does_not_fit_is_an_error_of_the_call():
    """A table of 2^29 tokens without max_len asks for 275 GB of logits."""
    k = torch.zeros(2, 8, 16, 64, dtype=BF, device=DEV)
    bt = torch.zeros(1, 1 << 25, dtype=torch.int32, device=DEV)
    q = torch.ones(1, 128, 64, dtype=BF, device=DEV)
    sc = torch.zeros(2, 8, 16, device=DEV)
    with pytest.raises(torch.OutOfMemoryError):
        ops.attention_decode_scored(q, torch.empty_like(q), k, k, bt, i32([20]), 1.0, sc)
    out = ops.attention_decode_scored(q, torch.empty_like(q), k, k, bt, i32([20]), 1.0, sc, max_len=32)
    assert out.abs().max() == 0 and (sc[0, :, :4].sum() > 0)


def test_calls_without_work():
    k = torch.zeros(2, 2, 16, 64, dtype=BF, device=DEV)
    sc, ps = torch.zeros(2, 2, 16, device=DEV), torch.zeros(2, 2, 16, dtype=torch.int32, device=DEV)
    bt, e = torch.zeros(0, 3, dtype=torch.int32, device=DEV), i32([])
    q = torch.zeros(0, 4, 64, dtype=BF, device=DEV)
    assert ops.attention_decode_scored(q, q.clone(), k, k, bt, e, 1.0, sc).shape == q.shape
    assert ops.kv_evict(k, k.clone(), sc, ps, bt, e, e, 4, 1).numel() == 0
