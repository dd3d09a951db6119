"""What the plain C launchers of the cache-budget kernels refuse before any
launch: they are usable without the torch binding, whose checks are then not
there. The pointers are never followed: every call here ends in a refusal."""
import ctypes

import pytest

from sched_pass_b200 import _build
from sched_pass_b200._ext import ext

P, I, L, F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float
REFUSED, NO_SCRATCH = -1, -2
AT = 1 << 20  # of the made-up addresses: 1 MB apart


class QkNormArgs(ctypes.Structure):
    _fields_ = [("qkv", P), ("ld_qkv", L), ("wq", P), ("wk", P), ("eps", F), ("pos", P), ("slot", P), ("cos_sin", P),
                ("max_pos", I), ("rot", I), ("q_out", P), ("ld_q", L), ("k_cache", P), ("v_cache", P), ("scores", P),
                ("positions", P), ("T", I), ("Hq", I), ("Hkv", I), ("D", I), ("page_size", I), ("num_pages", I),
                ("element", I), ("num_sms", I), ("status", P)]


class ScoredArgs(ctypes.Structure):
    _fields_ = [("q", P), ("q_req", L), ("q_query", L), ("out", P), ("out_req", L), ("out_query", L), ("lse", P),
                ("k_cache", P), ("v_cache", P), ("scores", P), ("block_table", P), ("bt_stride", L), ("bt_pages", I),
                ("kv_lens", P), ("R", I), ("Q", I), ("Hq", I), ("Hkv", I), ("D", I), ("page_size", I), ("num_pages", I),
                ("max_len", I), ("element", I), ("num_sms", I), ("sm_scale", F), ("ws", P), ("ws_floats", L), ("status", P)]


class KvEvictArgs(ctypes.Structure):
    _fields_ = [("k_cache", P), ("v_cache", P), ("scores", P), ("positions", P), ("block_table", P), ("bt_stride", L),
                ("bt_pages", I), ("kv_lens", P), ("last_pos", P), ("new_lens", P), ("R", I), ("Hkv", I), ("D", I),
                ("page_size", I), ("num_pages", I), ("max_len", I), ("budget", I), ("recent", I), ("sink", I),
                ("num_sms", I), ("ws", P), ("ws_ints", L), ("status", P)]


@pytest.fixture(scope="module")
def lib():
    ext()
    so = ctypes.CDLL(_build.ext_path())
    for name, args in (("sched_qk_norm_rope_kv_append", QkNormArgs), ("sched_attn_scored", ScoredArgs),
                       ("sched_kv_evict", KvEvictArgs)):
        getattr(so, name).argtypes = [ctypes.POINTER(args), P]
        getattr(so, name).restype = I
    so.sched_attn_scored_ws_floats.argtypes, so.sched_attn_scored_ws_floats.restype = [I] * 7, L
    so.sched_kv_evict_ws_ints.argtypes, so.sched_kv_evict_ws_ints.restype = [I] * 5, L
    return so


def addresses(names):
    return {n: AT * (i + 1) for i, n in enumerate(names)}


def append(lib, **change):
    a = dict(addresses(["qkv", "wq", "wk", "pos", "slot", "cos_sin", "q_out", "k_cache", "v_cache"]), ld_qkv=512, ld_q=256,
             max_pos=16, rot=64, T=2, Hq=4, Hkv=2, D=64, page_size=16, num_pages=4, num_sms=148)
    a.update(change)
    return lib.sched_qk_norm_rope_kv_append(ctypes.byref(QkNormArgs(**a)), None)


def scored(lib, **change):
    """A call that needs scratch (heads of a window of 40 rows) and has none."""
    a = dict(addresses(["q", "out", "k_cache", "v_cache", "scores", "block_table", "kv_lens"]), q_req=5120, q_query=512,
             out_req=5120, out_query=512, bt_stride=4, bt_pages=4, R=2, Q=10, Hq=8, Hkv=2, D=64, page_size=16, num_pages=9,
             max_len=64, num_sms=148, sm_scale=0.125)
    a.update(change)
    return lib.sched_attn_scored(ctypes.byref(ScoredArgs(**a)), None)


def evict(lib, **change):
    """A call that needs scratch (a context whose keys shared memory does not hold) and has none."""
    a = dict(addresses(["k_cache", "v_cache", "scores", "positions", "block_table", "kv_lens", "last_pos", "new_lens"]),
             bt_stride=3000, bt_pages=3000, R=2, Hkv=2, D=64, page_size=16, num_pages=6000, max_len=48000, budget=100,
             recent=10, sink=2, num_sms=148)
    a.update(change)
    return lib.sched_kv_evict(ctypes.byref(KvEvictArgs(**a)), None)


@pytest.mark.parametrize("name", ["qkv", "wq", "wk", "pos", "slot", "cos_sin", "q_out", "k_cache", "v_cache"])
def test_append_refuses_missing_pointers(lib, name):
    assert append(lib, **{name: None}) == REFUSED


@pytest.mark.parametrize("change", [
    dict(num_sms=0), dict(ld_q=248), dict(ld_q=260), dict(ld_qkv=516), dict(q_out=AT + 8), dict(qkv=AT + 2), dict(D=96),
    dict(rot=24), dict(rot=80), dict(page_size=0), dict(num_pages=0), dict(max_pos=0), dict(Hq=0), dict(Hkv=0)])
def test_append_refuses(lib, change):
    assert append(lib, **change) == REFUSED


def test_scored_says_that_scratch_is_missing(lib):
    need = lib.sched_attn_scored_ws_floats(2, 10, 8, 2, 64, 64, 148)
    assert need > 0
    assert scored(lib) == NO_SCRATCH and scored(lib, ws=AT * 20, ws_floats=need - 1) == NO_SCRATCH


@pytest.mark.parametrize("change", [
    dict(out=AT + 8), dict(out=AT + 2), dict(out_req=5124), dict(out_query=260), dict(q=AT + 8), dict(q_req=4), dict(q_query=2),
    dict(k_cache=AT + 8), dict(v_cache=AT + 4), dict(scores=AT + 4), dict(ws=AT + 4, ws_floats=1 << 40), dict(num_sms=0),
    dict(Hq=7), dict(page_size=24), dict(bt_pages=0), dict(max_len=0), dict(D=32), dict(R=65536), dict(Q=8192)])
def test_scored_refuses(lib, change):
    assert scored(lib, **change) == REFUSED


@pytest.mark.parametrize("name", ["q", "out", "k_cache", "v_cache", "scores", "block_table", "kv_lens"])
def test_scored_refuses_missing_pointers(lib, name):
    assert scored(lib, **{name: None}) == REFUSED


def test_evict_says_that_scratch_is_missing(lib):
    need = lib.sched_kv_evict_ws_ints(2, 2, 48000, 100, 148)
    assert need > 0
    assert evict(lib) == NO_SCRATCH and evict(lib, ws=AT * 20, ws_ints=need - 1) == NO_SCRATCH
    # tracking tensors need no 16-byte boundary, nor do the lengths
    assert evict(lib, scores=AT + 4, positions=AT * 3 + 4, kv_lens=AT * 6 + 4) == NO_SCRATCH
    # lengths side by side are apart
    assert evict(lib, kv_lens=AT * 9, new_lens=AT * 9 + 8, last_pos=AT * 9 + 16) == NO_SCRATCH


@pytest.mark.parametrize("change", [
    dict(ws=AT * 20 + 4, ws_ints=1 << 40), dict(ws=AT * 20 + 8, ws_ints=1 << 40), dict(new_lens=AT * 6), dict(new_lens=AT * 7),
    dict(new_lens=AT * 6 + 4), dict(new_lens=AT * 7 - 4), dict(k_cache=AT + 8), dict(v_cache=AT + 2), dict(num_sms=0),
    dict(budget=0), dict(recent=99), dict(recent=-1), dict(sink=-1), dict(page_size=0), dict(bt_pages=0), dict(max_len=0),
    dict(D=96), dict(R=65536), dict(num_pages=1 << 30)])
def test_evict_refuses(lib, change):
    assert evict(lib, **change) == REFUSED


@pytest.mark.parametrize("name", ["k_cache", "v_cache", "scores", "positions", "block_table", "kv_lens", "last_pos", "new_lens"])
def test_evict_refuses_missing_pointers(lib, name):
    assert evict(lib, **{name: None}) == REFUSED


def test_calls_without_work_do_nothing(lib):
    assert append(lib, T=0) == 0 and scored(lib, R=0) == 0 and scored(lib, Q=0) == 0 and evict(lib, R=0) == 0


@pytest.mark.parametrize("R,Q,Hq,Hkv,D,max_len,kernels", [
    (3, 1, 8, 2, 128, 48, 1), (16, 1, 8, 2, 128, 224, 1), (2, 1, 8, 2, 128, 912, 1),      # short decode loops
    (4, 1, 8, 2, 128, 5008, 1), (200, 1, 8, 8, 64, 176, 1),
    (300, 1, 8, 2, 128, 224, 2), (1, 1, 32, 8, 128, 12000, 2), (40, 1, 32, 8, 128, 1664, 2),
    (64, 1, 32, 8, 128, 20000, 2), (2, 16, 8, 2, 128, 6000, 2)])
def test_form_of_a_scored_call(lib, R, Q, Hq, Hkv, D, max_len, kernels):
    """Which calls take one kernel (and no scratch) on 148 SMs: what the GPU
    tests of scratch, streams and graphs rely on."""
    assert (lib.sched_attn_scored_ws_floats(R, Q, Hq, Hkv, D, max_len, 148) > 0) == (kernels == 2)


@pytest.mark.parametrize("max_len,budget,scratch", [(40960, 100, False), (40961, 100, True), (224, 200, False), (50000, 50000, False)])
def test_evictions_that_need_scratch(lib, max_len, budget, scratch):
    assert (lib.sched_kv_evict_ws_ints(2, 1, max_len, budget, 148) > 0) == scratch
