"""Quantized KV caches on the GPU: append, read back, attention, and the fused norm + rotation + append, each against a plain
64-bit reference at the sizes, layouts and masks where it can go wrong."""
import ctypes as C

import numpy as np
import pytest

import oracle
from aion_b200 import capi
from aion_b200.backend import (AttentionWindow, BackendError, Chunk, DeviceStore, StepAttention, StepQKNormRopeAppend, StepRMSNorm,
                               StepRoPE1D, StepSequenceAppend, StepSequenceRead, TensorMeta)
from tests import kv_cache_ref as ref
from tests.kv_cache_ref import F16, F32, I32, Q4, Q8

pytestmark = pytest.mark.gpu
UNB = capi.WINDOW_UNBOUNDED
NAMES = {Q4: "q4", Q8: "q8", F16: "f16", F32: "f32"}


@pytest.fixture
def sess(backend):
    store = DeviceStore(backend.device_memory)
    s = backend.create_session(store)
    yield s, store
    backend.sync()
    store.deinit()


def put(store, arr, dtype, **kw):
    arr = np.ascontiguousarray(arr)
    return store.add(TensorMeta(dtype, arr.shape, **kw), arr)


def put_cache(store, stored, dtype, D, **kw):
    """A cache tensor from its stored rows [B, T, H, bytes or D]."""
    return store.add(TensorMeta(dtype, (*stored.shape[:3], D), quant_axis=3, **kw), np.ascontiguousarray(stored))


def read_bytes(store, tid, like):
    return store.read(tid).view(np.uint8).reshape(np.ascontiguousarray(like).view(np.uint8).shape)


# ---- append ---------------------------------------------------------------------------------
@pytest.mark.parametrize("H,D,Ln", [(1, 32, 1), (3, 32, 7), (2, 64, 1), (1, 96, 5), (4, 128, 33), (1, 256, 2)])
@pytest.mark.parametrize("src", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("dtype", [Q8, Q4], ids=["q8", "q4"])
@pytest.mark.parametrize("layout", ["plain", "paged", "rolling"])
def test_append_writes_the_blocks_of_the_quantizer(sess, layout, dtype, src, H, D, Ln):
    s, store = sess
    rng = np.random.default_rng([H, D, Ln, src, dtype])
    B, T = 3, 50
    new = (rng.standard_normal((B, Ln, H, D)) * rng.choice([1e-3, 1.0, 50.0], (B, Ln, H, 1))).astype(ref.NP[src])
    new[0, 0, 0, :32] = 0.0                              # a block of zeros
    cache = ref.pack(dtype, rng.standard_normal((B, T, H, D)).astype(np.float32))
    idx = np.array([0, T - Ln, 9], dtype=np.int32)
    if layout == "rolling":
        idx = np.array([0, T - 1, 4 * T + 13], dtype=np.int32)
    want = cache.copy()
    packed = ref.pack(dtype, new.astype(np.float32))
    for b in range(B):
        for t in range(Ln):
            want[b, (idx[b] + t) % T] = packed[b, t]
    table = None
    stored = cache
    if layout == "paged":
        stored, table = ref.to_pool(cache, 16, rng)
        full = stored.copy()
        for b in range(B):
            for t in range(T):
                full[table[b, t // 16], t % 16] = want[b, t]
        want = full
    tc = put_cache(store, stored, dtype, D, cache_policy="rolling" if layout == "rolling" else "none")
    tt = put(store, table, I32) if table is not None else None
    s.execute([StepSequenceAppend(cache=tc, new_kv=put(store, new, src), end_index=put(store, idx, I32), page_table=tt)])
    assert np.array_equal(read_bytes(store, tc, want), want.view(np.uint8))


def test_append_of_extreme_values_follows_the_quantizer(sess):
    """Subnormal, huge, infinite and NaN values: the same bytes as aion_cuda_quantize makes."""
    from aion_b200.backend import quantize
    s, store = sess
    rng = np.random.default_rng(5)
    rows = rng.standard_normal((1, 40, 1, 64)).astype(np.float32)
    rows *= np.float32(10.0) ** rng.integers(-38, 38, (1, 40, 1, 1)).astype(np.float32)
    rows[0, 3, 0, 5], rows[0, 4, 0, 6], rows[0, 5, 0, 7] = np.inf, np.nan, -np.inf
    rows[0, 6] = np.float32(0.5)                          # every value on a border of its own
    rows[0, 7, 0, :32] = (np.arange(32) - 16) / np.float32(2) * 7
    for dtype in (Q8, Q4):
        tc = put_cache(store, ref.pack(dtype, np.zeros((1, 40, 1, 64), np.float32)), dtype, 64)
        s.execute([StepSequenceAppend(cache=tc, new_kv=put(store, rows, F32), end_index=put(store, np.zeros(1, np.int32), I32))])
        want = quantize(s.backend, dtype, rows.reshape(40, 64), 1)
        assert np.array_equal(store.read(tc).view(np.uint8).reshape(-1), want)


@pytest.mark.parametrize("dtype", [Q8, Q4], ids=["q8", "q4"])
def test_a_ring_keeps_the_last_of_more_new_rows_than_it_holds(sess, dtype):
    s, store = sess
    rng = np.random.default_rng(6)
    new = rng.standard_normal((2, 37, 2, 64)).astype(np.float32)
    idx = np.array([3, 40], dtype=np.int32)
    tc = put_cache(store, ref.pack(dtype, np.zeros((2, 16, 2, 64), np.float32)), dtype, 64, cache_policy="rolling")
    s.execute([StepSequenceAppend(cache=tc, new_kv=put(store, new, F32), end_index=put(store, idx, I32))])
    want = np.empty((2, 16, 2, 64), np.float32)
    for b in range(2):
        for t in range(37):
            want[b, (idx[b] + t) % 16] = new[b, t]
    packed = ref.pack(dtype, want)
    assert np.array_equal(read_bytes(store, tc, packed), packed)


def test_append_reports_bad_ranges_and_pages_and_writes_nothing_of_them(sess, backend):
    s, store = sess
    rng = np.random.default_rng(7)
    cache = ref.pack(Q8, rng.standard_normal((3, 32, 1, 64)).astype(np.float32))
    new = rng.standard_normal((3, 4, 1, 64)).astype(np.float32)
    tn = put(store, new, F32)
    packed = ref.pack(Q8, new)
    tc = put_cache(store, cache, Q8, 64)
    s.execute([StepSequenceAppend(cache=tc, new_kv=tn, end_index=put(store, np.array([-1, 28, 29], np.int32), I32))])
    with pytest.raises(BackendError):
        backend.sync()
    want = cache.copy()
    want[1, 28:] = packed[1]
    assert np.array_equal(read_bytes(store, tc, want), want)
    pool, table = ref.to_pool(cache, 8, rng)
    table[0, 0], table[2, 0] = -1, pool.shape[0]
    tp = put_cache(store, pool, Q8, 64)
    s.execute([StepSequenceAppend(cache=tp, new_kv=tn, end_index=put(store, np.array([6, 0, 6], np.int32), I32), page_table=put(store, table, I32))])
    with pytest.raises(BackendError):
        backend.sync()
    want = pool.copy()
    want[table[0, 1], :2], want[table[1, 0], :4], want[table[2, 1], :2] = packed[0, 2:], packed[1], packed[2, 2:]
    assert np.array_equal(read_bytes(store, tp, want), want)


# ---- read -------------------------------------------------------------------------------------
@pytest.mark.parametrize("H,D", [(1, 32), (3, 32), (2, 64), (1, 96), (5, 128), (2, 256)])
@pytest.mark.parametrize("out", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("dtype", [Q8, Q4, F16, F32], ids=["q8", "q4", "f16", "f32"])
@pytest.mark.parametrize("layout", ["plain", "paged", "rolling"])
def test_read_gives_the_values_of_held_steps_and_zeros(sess, layout, dtype, out, H, D):
    s, store = sess
    rng = np.random.default_rng([H, D, out, dtype])
    B, T, Ln = 5, 45, 23
    cache = ref.pack(dtype, (rng.standard_normal((B, T, H, D)) * 3).astype(np.float32))
    start = np.array([0, 40, 7, 22, 44], dtype=np.int32)
    lens = np.array([0, T, 12, 45, 45], dtype=np.int32)
    if layout == "rolling":
        start = np.array([0, 100, 60, 2, 44], dtype=np.int32)
        lens = np.array([0, 118, 83, 20, 46], dtype=np.int32)
    vals = ref.unpack(dtype, cache).astype(np.float32)
    want = np.zeros((B, Ln, H, D), np.float32)
    for b in range(B):
        for t in range(Ln):
            step = start[b] + t
            if max(0, lens[b] - T) <= step < lens[b]:
                want[b, t] = vals[b, step % T]
    stored, tt = cache, None
    if layout == "paged":
        stored, table = ref.to_pool(cache, 16, rng)
        for b in range(B):  # pages without a step that is read are not looked up
            for i in range(table.shape[1]):
                if not any(i * 16 <= st < min(lens[b], i * 16 + 16) for st in range(start[b], start[b] + Ln)):
                    table[b, i] = -7
        tt = put(store, table, I32)
    tc = put_cache(store, stored, dtype, D, cache_policy="rolling" if layout == "rolling" else "none")
    to = store.add(TensorMeta(out, (B, Ln, H, D)), np.full((B, Ln, H, D), 9, ref.NP[out]))
    s.execute([StepSequenceRead(out=to, cache=tc, start_index=put(store, start, I32), lengths=put(store, lens, I32), page_table=tt)])
    assert np.array_equal(store.read(to), want.astype(ref.NP[out]))


def test_read_without_start_and_lengths_reads_the_whole_cache(sess):
    s, store = sess
    cache = ref.pack(Q4, np.random.default_rng(8).standard_normal((2, 19, 3, 64)).astype(np.float32))
    tc, to = put_cache(store, cache, Q4, 64), store.add(TensorMeta(F32, (2, 25, 3, 64)))
    s.execute([StepSequenceRead(out=to, cache=tc)])
    got = store.read(to)
    assert np.array_equal(got[:, :19], ref.unpack(Q4, cache).astype(np.float32)) and not got[:, 19:].any()


def test_read_reports_bad_starts_lengths_and_pages(sess, backend):
    s, store = sess
    rng = np.random.default_rng(9)
    cache = ref.pack(Q8, rng.standard_normal((4, 32, 1, 64)).astype(np.float32))
    vals = ref.unpack(Q8, cache).astype(np.float32)
    tc = put_cache(store, cache, Q8, 64)
    to = store.add(TensorMeta(F32, (4, 10, 1, 64)), np.full((4, 10, 1, 64), 5, np.float32))
    s.execute([StepSequenceRead(out=to, cache=tc, start_index=put(store, np.array([-1, 0, 0, 30], np.int32), I32),
                                lengths=put(store, np.array([32, -3, 33, 32], np.int32), I32))])
    with pytest.raises(BackendError):
        backend.sync()
    got = store.read(to)
    assert not got[:3].any() and np.array_equal(got[3, :2], vals[3, 30:]) and not got[3, 2:].any()
    pool, table = ref.to_pool(cache, 8, rng)
    table[1, 0], table[2, 1] = -1, pool.shape[0]
    s.execute([StepSequenceRead(out=to, cache=put_cache(store, pool, Q8, 64), page_table=put(store, table, I32))])
    with pytest.raises(BackendError):
        backend.sync()
    got = store.read(to)
    assert np.array_equal(got[0], vals[0, :10]) and not got[1, :8].any() and np.array_equal(got[1, 8:], vals[1, 8:10])
    assert np.array_equal(got[2, :8], vals[2, :8]) and not got[2, 8:].any()


@pytest.mark.parametrize("shift", [2, 4, 8, 18])
@pytest.mark.parametrize("dtype", [Q8, Q4], ids=["q8", "q4"])
def test_caches_at_any_even_address(sess, backend, dtype, shift):
    """A cache that begins `shift` bytes into an allocation: append, read and attention give the same as an aligned one."""
    s, store = sess
    rng = np.random.default_rng(shift)
    B, T, H, D = 2, 40, 2, 64
    cache = ref.pack(dtype, rng.standard_normal((B, T, H, D)).astype(np.float32))
    new = rng.standard_normal((B, 3, H, D)).astype(np.float32)
    idx = np.array([5, 30], dtype=np.int32)
    raw = store.add(TensorMeta(capi.DTYPE_I8, (cache.size + 64,)), np.concatenate([np.zeros(shift, np.uint8), cache.reshape(-1), np.zeros(64 - shift, np.uint8)]))
    ch = store.acquire_mut(raw)
    tc = store.bind(TensorMeta(dtype, (B, T, H, D), quant_axis=3), Chunk(ch.handle, shift, cache.size))
    to, ta = store.add(TensorMeta(F32, (B, T, H, D))), store.add(TensorMeta(F32, (B, 1, 4, D)))
    q = rng.standard_normal((B, 1, 4, D)).astype(np.float32)
    s.execute([StepSequenceAppend(cache=tc, new_kv=put(store, new, F32), end_index=put(store, idx, I32)), StepSequenceRead(out=to, cache=tc),
               StepAttention(out=ta, q=put(store, q, F32), k=tc, v=tc, scale=0.125)])
    for b in range(B):
        cache[b, idx[b]:idx[b] + 3] = ref.pack(dtype, new[b])
    assert np.array_equal(store.read(to), ref.unpack(dtype, cache).astype(np.float32))
    out = store.read(raw).view(np.uint8)
    assert not out[:shift].any() and not out[shift + cache.size:].any()
    want, bound = ref.attention(q, cache, cache, dtype, dtype, scale=0.125, positions=np.zeros((B, 1), int), lengths=[T] * B, right=UNB)
    assert (np.abs(store.read(ta) - want) <= bound).all()


# ---- attention -----------------------------------------------------------------------------------
def run_attention(sess, q, k, v, kdt, vdt, *, scale, positions=None, lengths=None, layout="plain", page=16, window=None, cap=0.0, flags=0,
                  seed=1, image=None, spoil_rows=True):
    """StepAttention over stored rows k, v [B, T, H, bytes]. Rows that a request does not hold are filled with NaN scales."""
    s, store = sess
    D = q.shape[-1]
    B, T = k.shape[:2]
    k, v = k.copy(), v.copy()
    if spoil_rows and lengths is not None and layout != "rolling":
        for b in range(B):
            k[b, max(0, lengths[b]):], v[b, max(0, lengths[b]):] = 0xFF, 0xFF
    tt = None
    if layout == "paged":
        rng = np.random.default_rng(seed)
        k, table = ref.to_pool(k, page, rng)
        v2 = np.full((k.shape[0], page, *v.shape[2:]), 0xFF, np.uint8)
        for b in range(B):
            for i in range(table.shape[1]):
                part = v[b, i * page:(i + 1) * page]
                v2[table[b, i], : part.shape[0]] = part
                if lengths is not None and i * page >= lengths[b]:
                    table[b, i] = -1     # entries past a request's length are not read
        v = v2
        tt = put(store, table, I32)
    policy = "rolling" if layout == "rolling" else "none"
    tk, tv = put_cache(store, k, kdt, D, cache_policy=policy), put_cache(store, v, vdt, D, cache_policy=policy)
    tq = put(store, q, F16 if q.dtype == np.float16 else F32)
    to = store.add(TensorMeta(F32, q.shape), np.full(q.shape, 777, np.float32))
    step = StepAttention(out=to, q=tq, k=tk, v=tv, scale=scale, window=window or AttentionWindow(), attn_logits_soft_cap=cap, page_table=tt, flags=flags,
                         query_positions=put(store, positions, I32) if positions is not None else None,
                         kv_lengths=put(store, np.asarray(lengths, np.int32), I32) if lengths is not None else None, image=image)
    s.execute([step])
    return store.read(to), step


def inputs(seed, B, T, H, D, L, Hq, kdt, vdt, qdt=np.float32, spread=1.0):
    rng = np.random.default_rng(seed)
    q = (rng.standard_normal((B, L, Hq, D)) * 1.3 * spread).astype(qdt)
    k = ref.pack(kdt, rng.standard_normal((B, T, H, D)).astype(np.float32))
    v = ref.pack(vdt, (rng.standard_normal((B, T, H, D)) * rng.choice([0.02, 0.8, 20.0], (1, 1, H, 1))).astype(np.float32))
    return q, k, v


def check(got, want, bound):
    assert np.isfinite(got).all()
    over = np.abs(got - want) - bound
    assert (over <= 0).all(), f"{(over > 0).sum()} of {over.size} beyond the bound, worst {np.abs(got - want)[over > 0].max():g} against {bound[over > 0].min():g}"
    norm = np.linalg.norm(want)
    if norm:
        # rms: a result is a sum of up to 1500 terms of either sign, 1/sqrt(1500) of the sum of their sizes, each off by a few 2^-24
        assert np.linalg.norm(got - want) <= 1e-5 * norm


ALL = [(Q8, Q8), (Q8, Q4), (Q4, Q8), (Q4, Q4)]


@pytest.mark.parametrize("kdt,vdt", ALL, ids=[f"{NAMES[a]}{NAMES[b]}" for a, b in ALL])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("qdt", [np.float32, np.float16], ids=["f32", "f16"])
def test_decode_lengths_from_none_to_many(sess, kdt, vdt, D, qdt):
    T, lens = 700, [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 333, 700]
    B = len(lens)
    q, k, v = inputs([D, kdt, vdt], B, T, 2, D, 1, 6, kdt, vdt, qdt)
    pos = np.maximum(np.array(lens)[:, None] - 1, 0).astype(np.int32)
    got, _ = run_attention(sess, q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, window=AttentionWindow.causal())
    want, bound = ref.attention(q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens)
    check(got, want, bound)
    assert not got[0].any()


@pytest.mark.parametrize("Hq,H", [(1, 1), (2, 1), (3, 1), (4, 1), (5, 1), (7, 1), (8, 1), (9, 1), (16, 1), (20, 2), (8, 8), (12, 4)])
@pytest.mark.parametrize("L", [1, 3])
def test_head_layouts(sess, Hq, H, L):
    B, T, D = 2, 150, 64
    q, k, v = inputs([Hq, H, L], B, T, H, D, L, Hq, Q8, Q4)
    lens = [150, 77]
    pos = np.array([[n - L + i for i in range(L)] for n in lens], dtype=np.int32)
    got, _ = run_attention(sess, q, k, v, Q8, Q4, scale=0.125, positions=pos, lengths=lens, window=AttentionWindow.causal())
    check(got, *ref.attention(q, k, v, Q8, Q4, scale=0.125, positions=pos, lengths=lens))


@pytest.mark.parametrize("page", [1, 5, 16, 48, 64, 100])
@pytest.mark.parametrize("D,kdt,vdt", [(64, Q4, Q4), (128, Q8, Q4), (256, Q4, Q8)])
def test_pages_that_end_anywhere(sess, page, D, kdt, vdt):
    B, T, L = 3, 210, 2
    q, k, v = inputs([page, D], B, T, 2, D, L, 8, kdt, vdt)
    lens = [210, 1, 101]
    pos = np.array([[max(0, n - L + i) for i in range(L)] for n in lens], dtype=np.int32)
    got, _ = run_attention(sess, q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, layout="paged", page=page, window=AttentionWindow.causal())
    check(got, *ref.attention(q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens))


@pytest.mark.parametrize("window", [dict(left=UNB, right=0), dict(left=20, right=0), dict(left=0, right=0), dict(left=33, right=5), dict(left=UNB, right=UNB),
                                    dict(left=16, right=0, chunk=24), dict(left=3, right=3)], ids=str)
@pytest.mark.parametrize("layout", ["plain", "rolling", "paged"])
@pytest.mark.parametrize("L", [1, 6, 19])
def test_windows_and_rings(sess, window, layout, L):
    B, T, H, D = 4, 80, 2, 64
    q, k, v = inputs([L], B, T, H, D, L, 4, Q4, Q8)
    lens = [300, 80, 95, 30] if layout == "rolling" else [80, 80, 41, 30]
    first = [n - L for n in lens]
    first[1] = 5                                           # earlier positions than the newest: some rows of a ring see nothing
    pos = np.array([[max(0, f) + i for i in range(L)] for f in first], dtype=np.int32)
    w = dict(chunk=0) | window
    got, _ = run_attention(sess, q, k, v, Q4, Q8, scale=0.125, positions=pos, lengths=lens, layout=layout, window=AttentionWindow(**w), cap=30.0)
    check(got, *ref.attention(q, k, v, Q4, Q8, scale=0.125, positions=pos, lengths=lens, rolling=layout == "rolling", cap=30.0, **w))


@pytest.mark.parametrize("L,Hq,H,D", [(2, 8, 1, 256), (5, 16, 4, 64), (13, 8, 4, 128), (40, 8, 1, 256), (64, 4, 4, 64), (77, 6, 2, 128), (130, 8, 4, 256)])
@pytest.mark.parametrize("kdt,vdt", ALL, ids=[f"{NAMES[a]}{NAMES[b]}" for a, b in ALL])
def test_several_rows_per_request(sess, L, Hq, H, D, kdt, vdt):
    B, T = 2, 290
    q, k, v = inputs([L, D, kdt, vdt], B, T, H, D, L, Hq, kdt, vdt)
    lens = [290, 140]
    pos = np.array([[n - L + i for i in range(L)] for n in lens], dtype=np.int32)
    got, _ = run_attention(sess, q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, window=AttentionWindow.causal())
    check(got, *ref.attention(q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens))


@pytest.mark.parametrize("D", [64, 256])
def test_prompts_without_positions_or_lengths(sess, D):
    """Positions default to the row, lengths to the cache."""
    B, T, L = 2, 33, 33
    q, k, v = inputs([D], B, T, 2, D, L, 4, Q8, Q8)
    got, _ = run_attention(sess, q, k, v, Q8, Q8, scale=D ** -0.5, window=AttentionWindow.causal())
    check(got, *ref.attention(q, k, v, Q8, Q8, scale=D ** -0.5, positions=np.tile(np.arange(L), (B, 1)), lengths=[T] * B))


@pytest.mark.parametrize("L", [1, 4])
@pytest.mark.parametrize("spread", [1e-6, 1.0, 300.0, 3e4])
def test_queries_and_values_of_any_size(sess, L, spread):
    """Queries up to beyond f16's range, values down to its smallest scales: the two-term products keep their precision."""
    B, T, H, D = 2, 100, 2, 128
    rng = np.random.default_rng(11)
    q = (rng.standard_normal((B, L, 8, D)) * spread).astype(np.float32)
    k = ref.pack(Q8, (rng.standard_normal((B, T, H, D)) / max(1.0, spread)).astype(np.float32))
    v = ref.pack(Q4, (rng.standard_normal((B, T, H, D)) * 10.0 ** rng.integers(-4, 4, (B, 1, H, 1))).astype(np.float32))
    lens = [100, 51]
    pos = np.array([[n - L + i for i in range(L)] for n in lens], dtype=np.int32)
    got, _ = run_attention(sess, q, k, v, Q8, Q4, scale=0.09, positions=pos, lengths=lens, window=AttentionWindow.causal())
    check(got, *ref.attention(q, k, v, Q8, Q4, scale=0.09, positions=pos, lengths=lens))


@pytest.mark.parametrize("bad", [np.nan, np.inf, 65504.0])
@pytest.mark.parametrize("D", [64, 96, 256])
def test_what_a_row_does_not_see_does_not_reach_it(sess, bad, D):
    """A key row of NaN, infinite or huge scales inside the cache: rows before it (causal) are those of a clean cache."""
    B, T, H, L = 1, 90, 1, 12
    q, k, v = inputs([3], B, T, H, D, L, 8, Q8, Q8)
    pos = np.arange(70, 70 + L, dtype=np.int32)[None]
    want, bound = ref.attention(q, k, v, Q8, Q8, scale=0.1, positions=pos, lengths=[T])
    bits = np.frombuffer(np.float16(bad).tobytes(), np.uint8)
    for c in (k, v):
        c.reshape(B, T, H, D // 32, 34)[0, 76, :, :, :2] = bits
    s, store = sess
    got, _ = run_attention(sess_quiet(sess), q, k, v, Q8, Q8, scale=0.1, positions=pos, lengths=[T], window=AttentionWindow.causal())
    check(got[:, :6], want[:, :6], bound[:, :6])


class sess_quiet(tuple):
    """A session whose reads do not raise on a reported fault (a NaN among the visible keys is reported like any NaN softmax)."""

    def __new__(cls, sess):
        s, store = sess

        class Store:
            def __getattr__(self, name):
                return getattr(store, name)

            @staticmethod
            def read(tid):
                try:
                    return store.read(tid)
                except BackendError:
                    return store.read(tid)
        return tuple.__new__(cls, (s, Store()))


def test_attention_reports_bad_lengths_positions_and_pages(sess, backend):
    s, store = sess
    q, k, v = inputs([4], 2, 40, 1, 64, 1, 4, Q8, Q4)
    pos = np.array([[39], [39]], dtype=np.int32)
    for kw in (dict(lengths=[40, -1], positions=pos), dict(lengths=[41, 40], positions=pos), dict(lengths=[40, 40], positions=np.array([[3], [-2]], np.int32))):
        with pytest.raises(BackendError):
            run_attention(sess, q, k, v, Q8, Q4, scale=0.1, spoil_rows=False, **kw)
    pool, table = ref.to_pool(k, 16, np.random.default_rng(1))
    vpool = ref.pack(Q4, np.ones((*pool.shape[:3], 64), np.float32))
    for wrong in (-1, pool.shape[0], 2 ** 31 - 1):
        t2 = table.copy()
        t2[1, 1] = wrong
        to = store.add(TensorMeta(F32, q.shape))
        s.execute([StepAttention(out=to, q=put(store, q, F32), k=put_cache(store, pool, Q8, 64), v=put_cache(store, vpool, Q4, 64), scale=0.1,
                                 page_table=put(store, t2, I32))])
        with pytest.raises(BackendError):
            backend.sync()
        assert np.isfinite(store.read(to)).all()           # its keys are left out
    got, _ = run_attention(sess, q, k, v, Q8, Q4, scale=0.1, lengths=[40, 40], positions=pos)   # and the device goes on
    check(got, *ref.attention(q, k, v, Q8, Q4, scale=0.1, positions=pos, lengths=[40, 40], right=UNB))


def test_attention_refuses_a_mix_and_odd_heads(sess):
    s, store = sess
    half = store.add(TensorMeta(F16, (1, 8, 1, 64)))
    quant = store.add(TensorMeta(Q8, (1, 8, 1, 64), quant_axis=3))
    q, out = store.add(TensorMeta(F32, (1, 1, 1, 64))), store.add(TensorMeta(F32, (1, 1, 1, 64)))
    for k, v in ((half, quant), (quant, half)):
        with pytest.raises(BackendError) as e:
            s.execute([StepAttention(out=out, q=q, k=k, v=v)])
        assert e.value.name == "Unsupported"


@pytest.mark.parametrize("L,D", [(1, 128), (1, 256), (9, 64), (40, 128)])
def test_the_same_call_gives_the_same_bits(sess, L, D):
    """Alone, repeated, and replayed from a recorded program whose two steps run in parallel lanes."""
    s, store = sess
    T, B = 900, 2
    q, k, v = inputs([L, D, 1], B, T, 2, D, L, 8, Q4, Q8)
    q2, k2, v2 = inputs([L, D, 2], B, T, 2, D, L, 8, Q4, Q8)
    pos = np.tile(np.arange(T - L, T, dtype=np.int32), (B, 1))
    kw = dict(scale=0.1, positions=pos, lengths=[T, T], window=AttentionWindow.causal())
    a, step = run_attention(sess, q, k, v, Q4, Q8, **kw)
    b, step2 = run_attention(sess, q2, k2, v2, Q4, Q8, **kw)
    prog = s.record([step, step2])
    try:
        for _ in range(3):
            for st in (step, step2):
                store.write(st.out, np.zeros(q.shape, np.float32))
            prog.launch()
            assert np.array_equal(store.read(step.out), a) and np.array_equal(store.read(step2.out), b)
    finally:
        prog.destroy()


def test_attention_on_a_stream_of_the_callers(sess, backend):
    import torch
    s, store = sess
    q, k, v = inputs([9], 2, 300, 2, 128, 1, 8, Q8, Q8)
    a, step = run_attention(sess, q, k, v, Q8, Q8, scale=0.1)
    stream = torch.cuda.Stream()
    backend.sync()
    backend.set_stream(stream.cuda_stream)
    try:
        store.write(step.out, np.zeros(q.shape, np.float32))
        s.execute([step])
        assert np.array_equal(store.read(step.out), a)
    finally:
        backend.sync()
        backend.set_stream(None)


def test_key_rows_beyond_four_gigabytes(sess, backend):
    """A pool whose byte offsets pass 2^32: the pages in use lie at its end."""
    import torch
    s, store = sess
    D, H, page = 256, 8, 64
    row = H * D // 32 * 34
    pages = (5 << 30) // (row * page)
    pool = torch.zeros(pages * page * row, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    tid = store.bind(TensorMeta(Q8, (pages, page, H, D), quant_axis=3), Chunk(pool.data_ptr(), 0, pool.numel()))
    rng = np.random.default_rng(2)
    new = rng.standard_normal((1, 100, H, D)).astype(np.float32)
    q = rng.standard_normal((1, 1, H, D)).astype(np.float32)
    tt = put(store, np.array([[pages - 1, pages - 3]], np.int32), I32)
    to, ta = store.add(TensorMeta(F32, (1, 100, H, D))), store.add(TensorMeta(F32, (1, 1, H, D)))
    s.execute([StepSequenceAppend(cache=tid, new_kv=put(store, new, F32), end_index=put(store, np.zeros(1, np.int32), I32), page_table=tt),
               StepSequenceRead(out=to, cache=tid, page_table=tt),
               StepAttention(out=ta, q=put(store, q, F32), k=tid, v=tid, scale=0.0625, kv_lengths=put(store, np.array([100], np.int32), I32), page_table=tt)])
    packed = ref.pack(Q8, new)
    assert np.array_equal(store.read(to), ref.unpack(Q8, packed).astype(np.float32))
    check(store.read(ta), *ref.attention(q, packed, packed, Q8, Q8, scale=0.0625, positions=[[0]], lengths=[100], right=UNB))


# ---- norm + rotation + append -----------------------------------------------------------------------
def dequantized_error_bound(dtype, exact, eps_value):
    """How far a stored value may be from the f64 value that it stands for, when the value handed to the cache was off by
    eps_value: half a step of the format, which is amax / 127 or amax / 7 of its block with the scale rounded to f16 (2^-11),
    and one step more where that moves a value over a border."""
    if dtype == F16:
        return np.abs(exact) * 2.0 ** -11 + 2.0 ** -25 + eps_value
    blocks = np.abs(exact).reshape(*exact.shape[:-1], -1, 32)
    steps = blocks.max(-1, keepdims=True) / (127 if dtype == Q8 else 7)
    # q4_0 divides by the unrounded scale and multiplies by the rounded one: 7 codes x 2^-11 of a step
    return np.broadcast_to(steps * (0.5 + 8 * 2.0 ** -11 if dtype == Q4 else 0.5 + 128 * 2.0 ** -11), blocks.shape).reshape(exact.shape) + 2 * eps_value


@pytest.mark.parametrize("kdt,vdt", [(F16, F16), (Q8, Q4), (Q4, Q8), (F16, Q4), (Q4, Q4)])
@pytest.mark.parametrize("B,L,Hq,H,D,prop", [(1, 1, 8, 1, 256, 1.0), (3, 5, 4, 2, 64, 0.5), (2, 1, 3, 3, 128, 1.0), (1, 33, 2, 1, 96, 0.3), (70, 1, 2, 1, 64, 0.0),
                                             (2, 7, 16, 8, 128, 1.0), (2, 3, 0, 2, 64, 1.0), (1, 2, 2, 1, 1024, 0.75), (1, 2, 4, 0, 64, 1.0)])
@pytest.mark.parametrize("layout", ["plain", "paged", "rolling"])
def test_norm_rope_append(sess, kdt, vdt, B, L, Hq, H, D, prop, layout):
    s, store = sess
    rng = np.random.default_rng([B, L, Hq, D, kdt, vdt])
    T, eps, base = L + 20, 1e-5, 10000.0
    stride = (Hq + 2 * H) * D + 12
    qkv = (rng.standard_normal((B, L, stride)) * rng.choice([0.01, 1.0, 30.0], (B, L, 1))).astype(np.float32)
    qg, kg = (1 + 0.3 * rng.standard_normal((2, D))).astype(np.float32)
    start = rng.integers(0, T - L + 1, B).astype(np.int32)
    if layout == "rolling":
        start = rng.integers(0, 5 * T, B).astype(np.int32)
    pos = (start[:, None] * 37 + np.arange(L)[None]).astype(np.int32)
    x = qkv[..., :(Hq + 2 * H) * D].reshape(B, L, Hq + 2 * H, D)
    want_q = ref.norm_rope(x[:, :, :Hq], qg, pos, eps, base, prop)
    want_k = ref.norm_rope(x[:, :, Hq:Hq + H], kg, pos, eps, base, prop)
    want_v = x[:, :, Hq + H:].astype(np.float64)
    zero = lambda dt: ref.pack(dt, np.zeros((B, T, H, D), np.float32))
    ck, cv, tt = zero(kdt), zero(vdt), None
    if layout == "paged":
        ck, table = ref.to_pool(ck, 8, rng)
        ck.view(np.uint8)[:] = 0
        cv = np.zeros((*ck.shape[:3], cv.shape[3]), cv.dtype)
        tt = put(store, table, I32)
    policy = "rolling" if layout == "rolling" else "none"
    tk, tv = put_cache(store, ck, kdt, D, cache_policy=policy), put_cache(store, cv, vdt, D, cache_policy=policy)
    tx = store.add(TensorMeta(F32, qkv.shape), qkv)
    view = store.bind(TensorMeta(F32, (B, L, (Hq + 2 * H) * D), row_stride=stride), store.acquire_const(tx))
    tq = store.add(TensorMeta(F32, (B, L, Hq, D)), np.full((B, L, Hq, D), 7, np.float32))
    s.execute([StepQKNormRopeAppend(q_out=tq, qkv=view, positions=put(store, pos, I32), end_index=put(store, start, I32), k_cache=tk, v_cache=tv,
                                    base_frequency=base, q_gamma=put(store, qg, F32), k_gamma=put(store, kg, F32), eps=eps, rope_proportion=prop,
                                    page_table=tt)])
    # two rounded products of the norm, its inverse root, cos / sin, two products and a sum: 8 roundings of at most the head's largest pair
    size = lambda w: 8 * 2.0 ** -24 * np.abs(w).max(-1, keepdims=True) * 2.0 if w.size else 0.0
    assert (np.abs(store.read(tq) - want_q) <= size(want_q)).all()
    if not H:
        return
    for tid, dt, want in ((tk, kdt, want_k), (tv, vdt, want_v)):
        stored = store.read(tid).view(np.uint8).reshape(*ck.shape[:3], -1)
        if dt == F16:
            stored = stored.view(np.float16)
        got = ref.unpack(dt, stored)
        touched = np.zeros(got.shape[:2], bool)
        for b in range(B):
            for l in range(L):
                step = start[b] + l
                at = (table[b, step // 8], step % 8) if layout == "paged" else (b, step % T)
                touched[at] = True
                err = np.abs(got[at] - want[b, l])
                assert (err <= dequantized_error_bound(dt, want[b, l], size(want[b, l]) if tid == tk else 0.0)).all()
                if tid == tv:
                    assert np.array_equal(stored[at], ref.pack(dt, x[b, l, Hq + H:]))   # no arithmetic: the quantizer's blocks
        assert not stored.view(np.uint8)[~touched].any() or dt != F16   # other rows stay as they were
        fresh = ref.pack(dt, np.zeros((1, 1, H, D), np.float32))[0, 0]
        if layout != "paged":
            assert all(np.array_equal(row, fresh) for row in stored[~touched])
        else:
            assert not stored.view(np.uint8)[~touched].any()


@pytest.mark.parametrize("gammas", ["none", "q", "k"])
def test_norm_rope_append_without_a_norm_equals_the_plain_steps(sess, gammas):
    """Without a gamma the heads are those of RoPE1D bit for bit; with one they agree with RMSNorm, then RoPE1D."""
    s, store = sess
    rng = np.random.default_rng(21)
    B, L, Hq, H, D, T = 2, 3, 4, 2, 64, 16
    qkv = rng.standard_normal((B, L, (Hq + 2 * H) * D)).astype(np.float32)
    x = qkv.reshape(B, L, Hq + 2 * H, D)
    g = (1 + 0.2 * rng.standard_normal(D)).astype(np.float32)
    start = np.array([2, 9], np.int32)
    pos = start[:, None] + np.arange(L, dtype=np.int32)[None]
    tg, tz = put(store, g, F32), put(store, np.zeros(D, np.float32), F32)
    tp, ti = put(store, pos, I32), put(store, start, I32)
    zeros = ref.pack(Q8, np.zeros((B, T, H, D), np.float32))
    tk, tv = put_cache(store, zeros, Q8, D), put_cache(store, zeros, Q8, D)
    tq = store.add(TensorMeta(F32, (B, L, Hq, D)))
    s.execute([StepQKNormRopeAppend(q_out=tq, qkv=put(store, qkv, F32), positions=tp, end_index=ti, k_cache=tk, v_cache=tv, base_frequency=1e4,
                                    q_gamma=tg if gammas == "q" else None, k_gamma=tg if gammas == "k" else None)])
    q1, k1 = put(store, x[:, :, :Hq], F32), put(store, x[:, :, Hq:Hq + H], F32)
    steps = [StepRMSNorm(out=t, x=t, gamma=tg, beta=tz, eps=1e-6) for t, on in ((q1, gammas == "q"), (k1, gammas == "k")) if on]
    rk, rv = put_cache(store, zeros, Q8, D), put_cache(store, zeros, Q8, D)
    s.execute(steps + [StepRoPE1D(out=t, x=t, positions=tp, base_frequency=1e4) for t in (q1, k1)] +
              [StepSequenceAppend(cache=rk, new_kv=k1, end_index=ti), StepSequenceAppend(cache=rv, new_kv=put(store, x[:, :, Hq + H:], F32), end_index=ti)])
    q_same, k_same = np.array_equal(store.read(tq), store.read(q1)), np.array_equal(store.read(tk), store.read(rk))
    assert np.array_equal(store.read(tv), store.read(rv))
    assert q_same if gammas != "q" else np.abs(store.read(tq) - store.read(q1)).max() <= 16 * 2.0 ** -24 * np.abs(store.read(q1)).max()
    assert k_same if gammas != "k" else np.mean(store.read(tk) != store.read(rk)) < 0.01


def test_norm_rope_append_reports_what_it_does_not_write(sess, backend):
    s, store = sess
    rng = np.random.default_rng(22)
    B, H, D, T = 4, 1, 64, 8
    qkv = rng.standard_normal((B, 2, 3 * D)).astype(np.float32)
    qkv[1, 0, D + 3] = np.nan                              # a key head that has no norm
    zeros = ref.pack(Q8, np.zeros((B, T, H, D), np.float32))
    tk, tv = put_cache(store, zeros, Q8, D), put_cache(store, zeros, Q8, D)
    tq = store.add(TensorMeta(F32, (B, 2, 1, D)), np.zeros((B, 2, 1, D), np.float32))
    tg = put(store, np.ones(D, np.float32), F32)
    s.execute([StepQKNormRopeAppend(q_out=tq, qkv=put(store, qkv, F32), positions=put(store, np.ones((B, 2), np.int32), I32),
                                    end_index=put(store, np.array([-1, 0, 7, 6], np.int32), I32), k_cache=tk, v_cache=tv, base_frequency=1e4,
                                    q_gamma=tg, k_gamma=tg)])
    with pytest.raises(BackendError):
        backend.sync()
    k, v = (store.read(t).reshape(zeros.shape) for t in (tk, tv))
    packed = ref.pack(Q8, qkv[:, :, 2 * D:].reshape(B, 2, 1, D))
    assert np.array_equal(k[0], zeros[0]) and np.array_equal(k[2], zeros[2]) and np.array_equal(v[0], zeros[0]) and np.array_equal(v[2], zeros[2])
    assert np.array_equal(k[1, 0], zeros[1, 0]) and not np.array_equal(k[1, 1], zeros[1, 1])
    assert np.array_equal(v[1, :2], packed[1]) and np.array_equal(v[3, 6:], packed[3])
    assert np.isfinite(store.read(tq)).all() and np.abs(store.read(tq)).min(axis=(1, 2, 3)).max() > 0


# ---- a run of them together ----------------------------------------------------------------------------
@pytest.mark.parametrize("kdt,vdt", [(Q8, Q8), (Q8, Q4), (Q4, Q4)])
@pytest.mark.parametrize("layout", ["plain", "paged", "rolling"])
def test_a_prompt_then_tokens_then_the_way_out(sess, kdt, vdt, layout):
    """A prompt of 21 rows and three single tokens go through the fused step and attention; what attention saw is read back, and the
    attention of every step is that of the values read back."""
    s, store = sess
    rng = np.random.default_rng(31)
    B, Hq, H, D, T = 2, 8, 2, 128, 32
    policy = "rolling" if layout == "rolling" else "none"
    shape = (B, T) if layout != "paged" else (B * 4 + 1, 8)
    table = rng.permutation(B * 4 + 1)[: B * 4].reshape(B, 4).astype(np.int32)
    tt = put(store, table, I32) if layout == "paged" else None
    zk, zv = (ref.pack(dt, np.zeros((*shape, H, D), np.float32)) for dt in (kdt, vdt))
    tk, tv = put_cache(store, zk, kdt, D, cache_policy=policy), put_cache(store, zv, vdt, D, cache_policy=policy)
    tg = put(store, (1 + 0.2 * rng.standard_normal(D)).astype(np.float32), F32)
    done = 17 if layout == "rolling" else 0
    for n in (21, 1, 1, 1):
        pos = np.tile(done + np.arange(n, dtype=np.int32), (B, 1))
        lens = np.full(B, done + n, np.int32)
        tq, to = store.add(TensorMeta(F32, (B, n, Hq, D))), store.add(TensorMeta(F32, (B, n, Hq, D)))
        tp, tl = put(store, pos, I32), put(store, lens, I32)
        lo = max(0, done + n - T) if layout == "rolling" else 0
        held = done + n - lo
        fk, fv = store.add(TensorMeta(F32, (B, held, H, D))), store.add(TensorMeta(F32, (B, held, H, D)))
        ts = put(store, np.full(B, lo, np.int32), I32)
        s.execute([StepQKNormRopeAppend(q_out=tq, qkv=put(store, rng.standard_normal((B, n, (Hq + 2 * H) * D)).astype(np.float32), F32), positions=tp,
                                        end_index=put(store, np.full(B, done, np.int32), I32), k_cache=tk, v_cache=tv, base_frequency=1e4, q_gamma=tg,
                                        k_gamma=tg, page_table=tt),
                   StepAttention(out=to, q=tq, k=tk, v=tv, query_positions=tp, kv_lengths=tl, scale=0.088, window=AttentionWindow.causal(), page_table=tt),
                   StepSequenceRead(out=fk, cache=tk, start_index=ts, lengths=tl, page_table=tt),
                   StepSequenceRead(out=fv, cache=tv, start_index=ts, lengths=tl, page_table=tt)])
        k, v, q = store.read(fk), store.read(fv), store.read(tq)
        want, bound = ref.attention(q, k, v, F32, F32, scale=0.088, positions=pos - lo, lengths=[held] * B)
        check(store.read(to), want, bound)
        done += n


def test_an_expired_wait_is_reported_and_the_device_stays_usable(sess, backend):
    """The kernel's copy barriers time out instead of hanging: with the test hook every warp leaves out its first copy."""
    s, store = sess
    q, k, v = inputs([12], 2, 200, 1, 128, 1, 8, Q8, Q8)
    q, k, v = q, np.repeat(k, 2, 2), np.repeat(v, 2, 2)      # two kv heads: rows on 16-byte boundaries
    want, step = run_attention(sess, q, k, v, Q8, Q8, scale=0.1)
    lib = backend._lib
    assert lib.aion_cuda_debug_expire_waits(backend.handle, 1) == capi.OK
    try:
        s.execute([step])
        with pytest.raises(BackendError) as e:
            backend.sync()
        assert e.value.name == "ExecutionFailed"
    finally:
        lib.aion_cuda_debug_expire_waits(backend.handle, 0)
    s.execute([step])
    assert np.array_equal(store.read(step.out), want)


@pytest.mark.parametrize("layout,page,T", [("plain", 0, 96), ("rolling", 0, 96), ("rolling", 0, 90), ("paged", 32, 96), ("paged", 40, 96)])
@pytest.mark.parametrize("H", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("kdt,vdt", [(Q8, Q4), (Q4, Q8)])
def test_rows_on_and_off_sixteen_byte_boundaries(sess, layout, page, T, H, D, kdt, vdt):
    """Head counts and sizes whose rows begin on 16-byte boundaries and others, whole and ragged rings and pages."""
    B = 3
    q, k, v = inputs([H, D, T], B, T, H, D, 1, 2 * H, kdt, vdt)
    lens = [T + 37, T, 50] if layout == "rolling" else [T, 1, 50]
    pos = np.array([[n - 1] for n in lens], dtype=np.int32)
    got, _ = run_attention(sess, q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, layout=layout, page=page, window=AttentionWindow.causal())
    check(got, *ref.attention(q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, rolling=layout == "rolling"))


@pytest.mark.parametrize("dtype", [Q8, Q4], ids=["q8", "q4"])
def test_append_rounds_every_quotient_as_the_quantizer_does(sess, dtype):
    """Values on and beside the borders between codes, for many scales: every byte is the quantizer's."""
    from aion_b200.backend import quantize
    s, store = sess
    rng = np.random.default_rng(41)
    n = 20000
    top = (np.exp(rng.uniform(-6, 6, (n, 1))) * (1 + rng.integers(0, 2, (n, 1)))).astype(np.float32)
    levels = 127 if dtype == Q8 else 7
    scale = (top / np.float32(levels)).astype(np.float32)
    near = (rng.integers(-levels, levels, (n, 31)) + 0.5) * (scale.astype(np.float16).astype(np.float32) if dtype == Q8 else scale)
    near = near.astype(np.float32)
    near = (near.view(np.int32) + rng.integers(-2, 3, (n, 31), dtype=np.int32)).view(np.float32)   # up to two ulps off the border
    rows = np.concatenate([top, np.clip(near, -top, top)], 1).astype(np.float32)
    zeros = np.zeros((1, n, 1, 32 // 32 * (34 if dtype == Q8 else 18)), np.uint8)
    tc = put_cache(store, zeros, dtype, 32)
    s.execute([StepSequenceAppend(cache=tc, new_kv=put(store, rows.reshape(1, n, 1, 32), F32), end_index=put(store, np.zeros(1, np.int32), I32))])
    assert np.array_equal(store.read(tc).view(np.uint8).reshape(-1), quantize(s.backend, dtype, rows, 1))


FORCED = [capi.ATTENTION_ROW_UNITS, capi.ATTENTION_BLOCKS, capi.ATTENTION_GENERIC]


@pytest.mark.parametrize("flags", FORCED, ids=["columns", "rows", "any"])
@pytest.mark.parametrize("L,Hq,H,D", [(2, 8, 2, 256), (9, 14, 2, 64), (33, 8, 4, 128), (130, 2, 2, 64), (50, 6, 2, 256)])
@pytest.mark.parametrize("layout,page", [("plain", 0), ("paged", 24), ("rolling", 0)])
@pytest.mark.parametrize("kdt,vdt", ALL, ids=[f"{NAMES[a]}{NAMES[b]}" for a, b in ALL])
def test_each_kernel_on_several_rows(sess, flags, L, Hq, H, D, layout, page, kdt, vdt):
    """Causal rows with a window, in every layout, by each of the three kernels."""
    B, T = 2, 300
    q, k, v = inputs([L, D, kdt], B, T, H, D, L, Hq, kdt, vdt)
    lens = [711, 300] if layout == "rolling" else [300, 137]
    pos = np.array([[n - L + i for i in range(L)] for n in lens], dtype=np.int32)
    got, _ = run_attention(sess, q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, layout=layout, page=page,
                           window=AttentionWindow(left=150, right=0), cap=25.0, flags=flags)
    check(got, *ref.attention(q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, rolling=layout == "rolling", left=150, cap=25.0))


@pytest.mark.parametrize("flags", [capi.ATTENTION_ROW_UNITS, capi.ATTENTION_BLOCKS], ids=["columns", "rows"])
@pytest.mark.parametrize("L,T,kdt,vdt", [(7, 1400, Q8, Q4), (20, 1500, Q4, Q4), (3, 1100, Q8, Q8)])
def test_long_contexts_cut_over_clusters(sess, flags, L, T, kdt, vdt):
    """Few rows over many keys: the context is shared by the CTAs of a cluster, and one request has nothing."""
    B, H, D, Hq = 3, 1, 128, 4
    q, k, v = inputs([L, T], B, T, H, D, L, Hq, kdt, vdt)
    lens = [T, 0, T // 3]
    pos = np.array([[max(0, n - L) + i for i in range(L)] for n in lens], dtype=np.int32)
    got, _ = run_attention(sess, q, k, v, kdt, vdt, scale=0.1, positions=pos, lengths=lens, window=AttentionWindow.causal(), flags=flags)
    check(got, *ref.attention(q, k, v, kdt, vdt, scale=0.1, positions=pos, lengths=lens))
    assert not got[1].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("flags", [capi.ATTENTION_ROW_UNITS, capi.ATTENTION_BLOCKS], ids=["columns", "rows"])
def test_a_scale_that_is_not_finite_spoils_its_own_block(sess, bad, flags):
    """A V scale of NaN or infinity: the rows that see its key have NaN or infinities in the block's 32 dimensions, and their true
    values in the others; rows that do not see it are clean."""
    B, T, H, L, D = 1, 90, 1, 12, 128
    q, k, v = inputs([5], B, T, H, D, L, 4, Q8, Q4)
    pos = np.arange(70, 70 + L, dtype=np.int32)[None]
    kw = dict(scale=0.1, positions=pos, lengths=[T])
    want, bound = ref.attention(q, k, v, Q8, Q4, **kw)
    v.reshape(B, T, H, 4, 18)[0, 75, 0, 2, :2] = np.frombuffer(np.float16(bad).tobytes(), np.uint8)
    got, _ = run_attention(sess, q, k, v, Q8, Q4, window=AttentionWindow.causal(), flags=flags, **kw)
    clean = np.ones(got.shape, bool)
    clean[:, 5:, :, 64:96] = False
    assert not np.isfinite(got[~clean]).any()
    assert (np.abs(got - want)[clean] <= bound[clean]).all()


def test_an_expired_wait_in_the_rows_kernel_is_reported(sess, backend):
    s, store = sess
    q, k, v = inputs([13], 1, 200, 2, 128, 40, 4, Q8, Q8)
    want, step = run_attention(sess, q, k, v, Q8, Q8, scale=0.1, flags=capi.ATTENTION_BLOCKS)
    lib = backend._lib
    assert lib.aion_cuda_debug_expire_waits(backend.handle, 1) == capi.OK
    try:
        s.execute([step])
        with pytest.raises(BackendError) as e:
            backend.sync()
        assert e.value.name == "ExecutionFailed"
    finally:
        lib.aion_cuda_debug_expire_waits(backend.handle, 0)
    s.execute([step])
    assert np.array_equal(store.read(step.out), want)


# ---- the decoder ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("kdt,vdt,norm", [(Q8, Q8, False), (Q8, Q4, True), (Q4, Q4, True), (F16, F16, True)])
@pytest.mark.parametrize("R", [1, 5])
def test_decoder_with_quantized_caches_and_normed_heads(backend, R, kdt, vdt, norm, fused):
    """The synthetic decoder step by step against the same graph of oracle ops, and its recorded program against its steps. The
    chain re-quantizes its activations before every matmul: 2e-2, as for f16 caches (a code of the cache that falls on the other
    side of a border moves one value of 256 by a step, less than that)."""
    from aion_b200.decoder import DecoderConfig, SyntheticDecoder
    from oracle.decoder_ref import OracleDecoder
    from tests.test_gpu_decoder import CHAIN_TOL, make_values, rel_l2
    cfg = DecoderConfig(layers=2, hidden=256, ffn=512, heads=4, kv_heads=2, head_dim=64, vocab=512, ctx=32, k_dtype=kdt, v_dtype=vdt, qk_norm=norm)
    w, emb = make_values(cfg)
    dec = SyntheticDecoder(backend, cfg, R, lambda name, k, n: w[name], lambda v0, v1: emb[v0:v1], fused=fused)
    oracle_dec = OracleDecoder(cfg, R, w, emb)
    rng = np.random.default_rng(7)
    try:
        for t in range(4):
            tokens, pos = rng.integers(0, cfg.vocab, R).astype(np.int32), np.full(R, t, np.int32)
            dec.set_inputs(tokens, pos)
            dec.execute()
            _, logits, _ = oracle_dec.step(tokens, pos)
            got = dec.store.read(dec.logits).reshape(R, cfg.vocab)
            assert rel_l2(got, logits) < CHAIN_TOL
        dec.record()
        dec.launch()                                       # the last step again: the same row is written, the same keys are seen
        assert np.array_equal(dec.store.read(dec.logits).reshape(R, cfg.vocab), got)
    finally:
        dec.deinit()


@pytest.mark.parametrize("dtype", [Q8, Q4], ids=["q8", "q4"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_writes_the_image_of_its_output(sess, backend, dtype, D):
    """The activation image next to the output is the one that aion_cuda_act_image makes of it: alone and over a cluster."""
    from aion_b200.backend import act_image_meta
    from tests.gpu_util import DevBuf, make_image
    s, store = sess
    for T in (40, 1500):
        q, k, v = inputs([D, T], 3, T, 1, D, 1, 8, Q4, Q8)
        tid = store.add(act_image_meta(3, 8 * D, dtype))
        out, _ = run_attention(sess, q, k, v, Q4, Q8, scale=0.1, image=tid)
        buf = DevBuf(backend, np.ascontiguousarray(out, dtype=np.float32).reshape(-1))
        want = make_image(backend, dtype, buf, 3, 8 * D)
        assert np.array_equal(store.read(tid).view(np.uint8), want.read(np.uint8))
        buf.free(), want.free()


@pytest.mark.parametrize("T,L,first", [(1, 1, 7), (3, 2, 50), (5, 9, 2), (16, 4, 100), (17, 4, 2**31 - 21)])
def test_tiny_rings_and_steps_near_the_last(sess, T, L, first):
    """Rings of a few rows, and positions up to the largest 32-bit step."""
    B, H, D = 1, 2, 64
    q, k, v = inputs([T, L], B, T, H, D, L, 4, Q8, Q4)
    pos = first + np.arange(L, dtype=np.int64)[None]
    lens = [int(pos[0, -1]) + 1]
    for flags in (0, *FORCED):
        got, _ = run_attention(sess, q, k, v, Q8, Q4, scale=0.1, positions=pos.astype(np.int32), lengths=lens, layout="rolling",
                               window=AttentionWindow.causal(), flags=flags)
        check(got, *ref.attention(q, k, v, Q8, Q4, scale=0.1, positions=pos, lengths=lens, rolling=True))


@pytest.mark.parametrize("D,kdt,vdt", [(64, Q8, Q4), (128, Q4, Q4), (128, Q8, Q8), (256, Q4, Q8), (256, Q8, Q8)])
@pytest.mark.parametrize("layout,page", [("plain", 0), ("paged", 40), ("rolling", 0)])
def test_rows_kernel_over_many_stages(sess, D, kdt, vdt, layout, page):
    """As many units as SMs, so that a CTA walks a whole context of eleven stages alone: every ring of stages comes round."""
    B, T, H, L = 20, 700, 8, 2
    q, k, v = inputs([D, kdt, 5], B, T, H, D, L, H, kdt, vdt)
    lens = [T - 31 * b for b in range(B)]
    if layout == "rolling":
        lens = [n + 500 for n in lens]
    pos = np.array([[n - L + i for i in range(L)] for n in lens], dtype=np.int32)
    got, _ = run_attention(sess, q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, layout=layout, page=page,
                           window=AttentionWindow.causal(), flags=capi.ATTENTION_BLOCKS)
    check(got, *ref.attention(q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, rolling=layout == "rolling"))


def test_operands_that_overlap_are_refused(sess):
    """One cache for K and V, an output inside what is read."""
    s, store = sess
    cache, other = (put_cache(store, np.zeros((1, 8, 1, 2 * 34), np.uint8), Q8, 64) for _ in range(2))
    big = store.add(TensorMeta(F32, (1, 8, 1, 64)))
    qkv = put(store, np.zeros((1, 1, 192), np.float32), F32)
    q, pos, end = store.add(TensorMeta(F32, (1, 1, 1, 64))), put(store, np.zeros((1, 1), np.int32), I32), put(store, np.zeros(1, np.int32), I32)
    bind = lambda tid, meta: store.bind(meta, store.acquire_const(tid))
    rope = dict(q_out=q, qkv=qkv, positions=pos, end_index=end, k_cache=cache, v_cache=other, base_frequency=1e4)
    s.execute([StepQKNormRopeAppend(**rope)])
    for step in (StepQKNormRopeAppend(**{**rope, "v_cache": cache}), StepQKNormRopeAppend(**{**rope, "q_out": bind(qkv, TensorMeta(F32, (1, 1, 1, 64)))}),
                 StepSequenceRead(out=big, cache=bind(big, TensorMeta(Q8, (1, 8, 1, 64), quant_axis=3)))):
        with pytest.raises(BackendError) as e:
            s.execute([step])
        assert e.value.name == "InvalidArgument"


@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_scales_of_zero_and_below_are_refused(sess, scale):
    q, k, v = inputs([11], 2, 150, 1, 128, 3, 4, Q8, Q4)
    with pytest.raises(BackendError) as e:
        run_attention(sess, q, k, v, Q8, Q4, scale=scale)
    assert e.value.name == "InvalidArgument"


@pytest.mark.parametrize("bad", [np.nan, np.inf, 65504.0])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_what_a_row_of_a_block_does_not_see_does_not_reach_it(sess, bad, D):
    """The rows kernel: a K row of NaN, infinite or huge scales leaves the rows before it (causal) as they are."""
    B, T, H, L = 1, 90, 1, 12
    q, k, v = inputs([3], B, T, H, D, L, 8, Q8, Q8)
    pos = np.arange(70, 70 + L, dtype=np.int32)[None]
    want, bound = ref.attention(q, k, v, Q8, Q8, scale=0.1, positions=pos, lengths=[T])
    k.reshape(B, T, H, D // 32, 34)[0, 76, :, :, :2] = np.frombuffer(np.float16(bad).tobytes(), np.uint8)
    got, _ = run_attention(sess_quiet(sess), q, k, v, Q8, Q8, scale=0.1, positions=pos, lengths=[T], window=AttentionWindow.causal(), flags=capi.ATTENTION_BLOCKS)
    check(got[:, :6], want[:, :6], bound[:, :6])


def test_two_devices_of_one_gpu_at_once(sess, backend):
    """Two device objects, each with its stream and scratch, issue attention and appends in turn without waiting: both get what
    each gets alone."""
    from aion_b200.backend import CudaBackend
    other = CudaBackend(0)
    store2 = DeviceStore(other.device_memory)
    sess2 = (other.create_session(store2), store2)
    try:
        data = [inputs([n], 3, 1100, 2, 128, 1, 8, Q8, Q4) for n in (1, 2)]
        alone = [run_attention(x, *d, Q8, Q4, scale=0.1) for x, d in zip((sess, sess2), data)]
        for x, (_, step) in zip((sess, sess2), alone):
            x[1].write(step.out, np.zeros((3, 1, 8, 128), np.float32))
        for _ in range(20):
            for x, (_, step) in zip((sess, sess2), alone):
                x[0].execute([step])
        for x, (out, step) in zip((sess, sess2), alone):
            assert np.array_equal(x[1].read(step.out), out)
    finally:
        other.sync()
        store2.deinit()
        other.deinit()
