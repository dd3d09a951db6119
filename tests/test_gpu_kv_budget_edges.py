"""The cache-budget kernels where their arithmetic, scratch and scheduling can
go wrong: weights far below the largest, calls that need scratch on two streams
and in graphs, long runs of tiles, uneven batches.

Tolerances count roundings, as in test_gpu_kv_budget.py.
"""
import pytest
import torch

from sched_pass_b200 import _ext, ops
from sched_pass_b200.models import reference as ref
from test_gpu_kv_budget import (BF, DEV, FP, Budget, check_scored, evict_inputs, expect_bad_index, gen, i32, paged, randn, rope_table,
                                run_scored, scored_inputs)

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


# ------------------------------------------------------------------ the status words
def test_status_words_made_in_a_capture_outlive_replays(monkeypatch):
    """The first call that needs the status words is being captured: a replay
    neither erases what another call reported nor owns the words."""
    from sched_pass_b200.ops import kernels
    Hq, Hkv, D = 4, 2, 64
    g = gen(0)
    kc, vc = randn(g, 3, Hkv, 16, D, dtype=BF), randn(g, 3, Hkv, 16, D, dtype=BF)
    q, scores, bt, lens = randn(g, 1, Hq, D, dtype=BF), torch.zeros(3, Hkv, 16, device=DEV), i32([[2, 0]]), i32([20])
    out = torch.empty_like(q)
    qkv, w, cs = randn(g, 1, (Hq + 2 * Hkv) * D, dtype=BF), torch.ones(D, dtype=BF, device=DEV), rope_table(4, D)

    def attend():
        ops.attention_decode_scored(q, out, kc, vc, bt, lens, 0.1, scores)

    def append(slot):
        ops.qk_norm_rope_kv_append(qkv, w, w, 1e-5, i32([1]), slot, cs, q, kc, vc, Hq, Hkv)

    attend()  # lazy loading, before any capture
    append(i32([-1]))
    torch.cuda.synchronize()
    monkeypatch.setattr(kernels, "_status", {})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend()
    words = ops.status_buffer()
    assert words.tolist() == [0, 0, 0, 0]
    graph.replay()
    ops.check_status()
    append(i32([3 * 16 + 5]))  # a slot behind the cache
    graph.replay()
    expect_bad_index(3, 53)
    bt[0, 1] = -4
    graph.replay()
    expect_bad_index(8, -4)
    bt[0, 1] = 0
    append(i32([3 * 16 + 6]))
    torch.cuda.synchronize()
    del graph
    junk = [torch.full((4,), 7, dtype=torch.int32, device=DEV) for _ in range(64)]  # whoever takes over the graph's memory
    assert ops.status_buffer() is words and junk
    expect_bad_index(3, 54)


def test_status_words_of_another_stream_are_in_order(monkeypatch):
    """Made while their stream has work queued, used at once on another."""
    from sched_pass_b200.ops import kernels
    Hq, Hkv, D = 4, 2, 64
    kc = torch.zeros(3, Hkv, 16, D, dtype=BF, device=DEV)
    vc, q = torch.zeros_like(kc), torch.zeros(1, Hq, D, dtype=BF, device=DEV)
    qkv, w, cs = torch.ones(1, (Hq + 2 * Hkv) * D, dtype=BF, device=DEV), torch.ones(D, dtype=BF, device=DEV), rope_table(4, D)
    pos, slot = i32([1]), i32([48])
    big = torch.zeros(1 << 28, device=DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    monkeypatch.setattr(kernels, "_status", {})
    for _ in range(20):
        big.add_(1)
    ops.status_buffer()
    with torch.cuda.stream(side):
        ops.qk_norm_rope_kv_append(qkv, w, w, 1e-5, pos, slot, cs, q, kc, vc, Hq, Hkv)
    torch.cuda.synchronize()
    expect_bad_index(3, 48)


# ------------------------------------------------------------------ slots that an eviction freed
def test_evict_after_appends_that_start_no_tracking():
    """Tokens appended to freed slots by rope_kv_append: with the two
    assignments that kv_evict documents they are new tokens to the next
    eviction, and their entries are the old tokens' until then."""
    Hq, Hkv, D, budget, n = 4, 2, 128, 40, 64
    g = gen(8)
    bt, P = paged([n, n], 16)
    kc, vc, scores = randn(g, P, Hkv, 16, D, dtype=BF), randn(g, P, Hkv, 16, D, dtype=BF), torch.rand(P, Hkv, 16, generator=g, device=DEV)
    positions = torch.full((P, Hkv, 16), -1, dtype=torch.int32, device=DEV)
    positions[bt.long()] = torch.arange(n, dtype=torch.int32, device=DEV).view(1, 4, 1, 16).expand(2, 4, Hkv, 16)
    lens = ops.kv_evict(kc, vc, scores, positions, bt, i32([n, n]), i32([n - 1, n - 1]), budget, 8, sink=2)
    assert lens.tolist() == [budget] * 2
    cs, q = rope_table(n + 12, D), torch.empty(2, Hq, D, dtype=BF, device=DEV)
    for step in range(10):
        pos = i32([n + step] * 2)
        slot = bt[:, int(lens[0]) // 16] * 16 + lens % 16
        page, off = (slot // 16).long(), (slot % 16).long()
        stale = scores[page, :, off].clone(), positions[page, :, off].clone()
        ops.rope_kv_append(randn(g, 2, (Hq + 2 * Hkv) * D, dtype=BF), pos, slot, cs, q, kc, vc, Hq, Hkv)
        assert torch.equal(scores[page, :, off], stale[0]) and torch.equal(positions[page, :, off], stale[1])
        scores[slot // 16, :, slot % 16] = 0
        positions[slot // 16, :, slot % 16] = pos[:, None]
        lens = lens + 1
    state = [kc, vc, scores, positions]
    want = ref.kv_evict(*state, bt, lens, i32([n + 9] * 2), budget, 8, 2)
    got = ops.kv_evict(*state, bt, lens, i32([n + 9] * 2), budget, 8, sink=2)
    assert all(torch.equal(a, b) for a, b in zip((*state, got), want))
    for r in range(2):
        for h in range(Hkv):
            kept = positions[bt[r].long(), h].reshape(-1)[:budget].tolist()
            assert len(set(kept)) == budget and set(range(n + 2, n + 10)) | {0, 1} <= set(kept)


def test_scored_row_of_logits_that_are_all_minus_infinity():
    for lens in ([40, 17], [40, 17] + [0] * 300):  # one kernel, two kernels
        bt, P = paged(lens, 16)
        kc = torch.zeros(P, 2, 16, 64, dtype=BF, device=DEV)
        kc[..., 0] = -float("inf")
        vc, q = torch.ones_like(kc), torch.zeros(len(lens), 4, 64, dtype=BF, device=DEV)
        q[..., 0] = 1
        q[..., 1] = 1
        out, lse, scores = torch.full_like(q, 3.0), torch.zeros(len(lens), 4, device=DEV), torch.full((P, 2, 16), 0.5, device=DEV)
        ops.attention_decode_scored(q, out, kc, vc, bt, i32(lens), 1.0, scores, lse=lse)
        assert out.abs().max() == 0 and bool((lse == -float("inf")).all()) and bool((scores == 0.5).all())


# ------------------------------------------------------------------ the two-kernel form and its scratch
@pytest.mark.parametrize("lens,Q,Hq,Hkv,D,dtype", [
    ([12000], 1, 32, 8, 128, BF),                                # hundreds of partial results per row
    ([1664 - 29 * (i % 5) for i in range(40)], 1, 32, 8, 128, BF),  # runs of many tiles over requests and heads
    ([1500 - 31 * (i % 7) for i in range(70)], 1, 16, 4, 64, FP),
    ([20000] + [40 + i % 9 for i in range(63)], 1, 32, 8, 128, BF),  # one long request among many short ones
    ([9000, 3] + [17] * 98, 1, 16, 8, 64, FP),
    ([6000, 800], 16, 8, 2, 128, BF),                            # a long window: 64 query rows
    ([1800, 20000], 1, 64, 4, 128, FP)])                         # 16 query rows
def test_scored_long_runs_and_uneven_batches(lens, Q, Hq, Hkv, D, dtype):
    n0 = _ext.launches()
    run_scored(lens, Q, Hq, Hkv, D, dtype, seed=len(lens))
    assert _ext.launches() - n0 == 2


@pytest.mark.parametrize("lens,Q,Hq,Hkv,D", [
    ([1664 - 29 * (i % 5) for i in range(40)], 1, 32, 8, 128), ([900, 333, 2000], 5, 16, 2, 128), ([12000, 1], 1, 8, 8, 64)])
def test_scored_two_kernels_repeat_bit_for_bit(lens, Q, Hq, Hkv, D):
    q, kc, vc, bt, kl, scores0 = scored_inputs(lens, Q, Hq, Hkv, D, BF)
    res, n0 = [], _ext.launches()
    for i in range(5):
        scores, out, lse = scores0.clone(), torch.empty_like(q), torch.empty(q.shape[:3], device=DEV)
        junk = torch.full((1 << 22,), float("nan"), device=DEV)  # what the scratch holds before the call does not matter
        del junk
        ops.attention_decode_scored(q, out, kc, vc, bt, kl, 0.09, scores, lse=lse)
        res.append((out, scores, lse))
    assert _ext.launches() - n0 == 10
    assert all(torch.equal(a, b) for x in res[1:] for a, b in zip(x, res[0]))


def full_budget(seed, **kw):
    """A Budget whose caches are full up to a few tokens below the budget, of
    so many heads that the attention takes two kernels."""
    b = Budget(seed=seed, R=300, budget=200, slack=24, **kw)
    g = gen(seed + 100)
    for t in (b.kc, b.vc):
        t.copy_(randn(g, *t.shape))
    b.scores.copy_(torch.rand(b.scores.shape, generator=g, device=DEV))
    cols = b.bt.shape[1]
    at = torch.arange(cols * 16, dtype=torch.int32, device=DEV).view(1, cols, 1, 16).expand(b.R, cols, b.Hkv, 16)
    b.positions[b.bt.long()] = at
    b.lens.copy_(190 + torch.arange(b.R, device=DEV) % 20)
    b.pos.copy_(b.lens)
    return b


def same_budgets(x, y):
    return torch.equal(x.out, y.out) and torch.equal(x.lens, y.lens) and all(torch.equal(s, t) for s, t in zip(x.state(), y.state()))


def test_two_streams_with_scratch():
    """As test_two_streams_at_once, where the attention needs scratch and every step evicts."""
    pair, alone = [full_budget(s) for s in (1, 2)], [full_budget(s) for s in (1, 2)]
    start = [x.positions.clone() for x in pair]
    rows = randn(gen(4), 25, *pair[0].qkv.shape, dtype=BF)
    streams = [torch.cuda.Stream() for _ in pair]
    torch.cuda.synchronize()
    n0 = _ext.launches()
    for i in range(25):
        for x, st in zip(pair, streams):
            with torch.cuda.stream(st):
                x.qkv.copy_(rows[i])
                x.step()
    assert _ext.launches() - n0 == 25 * 2 * 4  # append, two of the attention, eviction
    torch.cuda.synchronize()
    for i in range(25):
        for x in alone:
            x.qkv.copy_(rows[i])
            x.step()
    for x, y, p in zip(pair, alone, start):
        assert same_budgets(x, y) and bool((x.lens == 200).all())
        assert not torch.equal(x.positions, p)


def test_captured_steps_with_scratch():
    """Two graphs whose calls have scratch, replayed at once on two streams
    with new inputs, beside eager copies."""
    graphed, eager = [full_budget(s) for s in (5, 6)], [full_budget(s) for s in (5, 6)]
    graphs, streams = [], [torch.cuda.Stream() for _ in graphed]
    for x in graphed:
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        n0 = _ext.launches()
        with torch.cuda.graph(gr):
            x.step()
        assert _ext.launches() - n0 == 4
        graphs.append(gr)
    rows = randn(gen(3), 20, *eager[0].qkv.shape, dtype=BF)
    torch.cuda.synchronize()
    for i in range(20):
        for x, gr, st in zip(graphed, graphs, streams):
            with torch.cuda.stream(st):
                x.qkv.copy_(rows[i])
                gr.replay()
    torch.cuda.synchronize()
    for i in range(20):
        for x in eager:
            x.qkv.copy_(rows[i])
            x.step()
    assert all(same_budgets(x, y) for x, y in zip(graphed, eager))


def test_evict_with_scratch_on_two_streams_and_in_graphs():
    """Contexts whose keys shared memory does not hold: eager on two streams at
    once, then two graphs at once, against the oracle."""
    cases = [([45001, 41000], 2000, 100), ([43777, 50000], 41000, 3)]
    states = [evict_inputs(lens, 1, 64, BF, seed=i) for i, (lens, _, _) in enumerate(cases)]
    want = [ref.kv_evict(*s, b, rec, 4) for s, (_, b, rec) in zip(states, cases)]
    work = [[t.clone() for t in s] for s in states]
    streams = [torch.cuda.Stream() for _ in cases]
    lens = [torch.empty_like(s[5]) for s in states]

    def evict(i):
        for t, s in zip(work[i][:4], states[i][:4]):
            t.copy_(s)
        ops.kv_evict(*work[i], cases[i][1], cases[i][2], sink=4, new_lens=lens[i])

    def check():
        torch.cuda.synchronize()
        for i, w in enumerate(want):
            assert all(torch.equal(a, b) for a, b in zip((*work[i][:4], lens[i]), w))
            for t in work[i][:4]:
                t.zero_()
            lens[i].zero_()
        torch.cuda.synchronize()

    torch.cuda.synchronize()
    for _ in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                for _ in range(4):
                    evict(i)
        check()
    graphs = []
    for i in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            evict(i)
        graphs.append(gr)
    for _ in range(3):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                for _ in range(4):
                    gr.replay()
        check()


# ------------------------------------------------------------------ outputs in place, long caches
@pytest.mark.parametrize("T", [3, 900, 4200])
def test_append_into_the_rows_that_it_reads(T):
    """q_out as a view of the projection's own rows: the query heads turn in place."""
    Hq, Hkv, D = 12, 4, 128
    g = gen(T)
    rows = randn(g, T, (Hq + 2 * Hkv) * D, dtype=BF)
    wq, wk = (1 + 0.2 * randn(g, D)).to(BF), (1 + 0.2 * randn(g, D)).to(BF)
    pos = torch.randint(0, 64, (T,), generator=g, device=DEV).to(torch.int32)
    slot = torch.randperm(T + 7, generator=g, device=DEV)[:T].to(torch.int32)
    P, cs = -(-(T + 7) // 16), rope_table(64, D)
    caches = [torch.zeros(P, Hkv, 16, D, dtype=BF, device=DEV) for _ in range(4)]
    q = torch.empty(T, Hq, D, dtype=BF, device=DEV)
    ops.qk_norm_rope_kv_append(rows, wq, wk, 1e-5, pos, slot, cs, q, *caches[:2], Hq, Hkv)
    own = rows.clone()
    ops.qk_norm_rope_kv_append(own, wq, wk, 1e-5, pos, slot, cs, own[:, :Hq * D].view(T, Hq, D), *caches[2:], Hq, Hkv)
    assert torch.equal(own[:, :Hq * D].view(T, Hq, D), q) and torch.equal(own[:, Hq * D:], rows[:, Hq * D:])
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


@pytest.mark.parametrize("lens,Q,Hq,Hkv,D", [([700, 33], 1, 8, 2, 128), ([1600] * 40, 1, 32, 8, 64), ([300, 2000] * 9, 6, 16, 2, 128)])
def test_scored_output_over_its_queries(lens, Q, Hq, Hkv, D):
    q, kc, vc, bt, kl, scores0 = scored_inputs(lens, Q, Hq, Hkv, D, BF)
    want, s1, s2 = torch.empty_like(q), scores0.clone(), scores0.clone()
    ops.attention_decode_scored(q, want, kc, vc, bt, kl, D**-0.5, s1)
    ops.attention_decode_scored(q, q, kc, vc, bt, kl, D**-0.5, s2)
    assert torch.equal(q, want) and torch.equal(s1, s2)


def test_scored_two_kernels_with_offsets_past_32_bits():
    P, Hkv, D, n = 270000, 8, 128, 3000
    kc = torch.empty(P, Hkv, 16, D, dtype=BF, device=DEV)
    vc, scores = torch.empty_like(kc), torch.zeros(P, Hkv, 16, device=DEV)
    last = P - 1 - torch.randperm(188, generator=gen(1), device=DEV)
    g = gen(2)
    kc[last], vc[last] = randn(g, 188, Hkv, 16, D, dtype=BF), randn(g, 188, Hkv, 16, D, dtype=BF)
    small = kc[last].clone(), vc[last].clone()
    table = torch.zeros(60, 188, dtype=torch.int32, device=DEV)
    table[7] = last.to(torch.int32)
    lens = i32([0] * 7 + [n] + [0] * 52)
    q = randn(g, 60, 1, 16, D, dtype=BF)
    out, n0 = torch.empty_like(q), _ext.launches()
    ops.attention_decode_scored(q, out, kc, vc, table, lens, D**-0.5, scores)
    assert _ext.launches() - n0 == 2
    check_scored(q[7:8], *small, torch.arange(188, dtype=torch.int32, device=DEV)[None], i32([n]),
                 torch.zeros(188, Hkv, 16, device=DEV), out[7:8], None, scores[last], D**-0.5)
    assert out[:7].abs().max() == 0 and out[8:].abs().max() == 0
