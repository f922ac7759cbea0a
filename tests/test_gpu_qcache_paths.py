"""Attention over quantized caches: every path of its kernels, each test sure of the kernel that it ran."""
import ctypes as C

import numpy as np
import pytest

from aion_b200 import capi
from aion_b200.backend import AttentionWindow
from tests import kv_cache_ref as ref
from tests.kv_cache_ref import Q4, Q8
from tests.test_gpu_kv_cache import ALL, NAMES, inputs, run_attention, sess, sess_quiet  # noqa: F401

pytestmark = pytest.mark.gpu
ROWS, COLUMNS, BOXES, ANY = capi.QCACHE_KERNEL_ROWS, capi.QCACHE_KERNEL_COLUMNS, capi.QCACHE_KERNEL_COLUMNS_BOXES, capi.QCACHE_KERNEL_ANY
IDS = [f"{NAMES[a]}{NAMES[b]}" for a, b in ALL]


def launched(backend):
    """(kernel, CTAs of a cluster, dealt) of the last attention."""
    v = [C.c_uint32() for _ in range(3)]
    assert backend._lib.aion_cuda_debug_qcache_kernel(backend.handle, *(C.byref(x) for x in v)) == capi.OK
    return tuple(x.value for x in v)


def within(got, want, bound):
    """No further from the 64-bit result than f32 arithmetic may be (kv_cache_ref.attention)."""
    assert np.isfinite(got).all()
    over = np.abs(got - want) - bound
    assert (over <= 0).all(), f"{(over > 0).sum()} of {over.size} beyond the bound, worst by {over.max():g}"


def causal(lens, L):
    return np.array([[max(0, n - L) + i for i in range(L)] for n in lens], dtype=np.int32)


@pytest.mark.parametrize("kdt,vdt", ALL, ids=IDS)
@pytest.mark.parametrize("D,H,Hq", [(64, 4, 8), (128, 2, 8), (256, 1, 4)])
@pytest.mark.parametrize("layout,page", [("plain", 0), ("paged", 40), ("rolling", 0)])
@pytest.mark.parametrize("L,T,cluster", [(20, 600, 2), (7, 1100, 4), (3, 2100, 8)])
def test_rows_share_the_keys_of_a_cluster(sess, backend, kdt, vdt, D, H, Hq, layout, page, L, T, cluster):
    """Few blocks of rows over many keys: the CTAs of a cluster add up their sums; one request has no keys, and one so few that
    most of its CTAs have none."""
    lens = [T, 0, 70] if layout != "rolling" else [3 * T + 5, 0, 70]
    B = len(lens)
    q, k, v = inputs([D, L, kdt], B, T, H, D, L, Hq, kdt, vdt)
    pos = causal(lens, L)
    got, _ = run_attention(sess, q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, layout=layout, page=page,
                           window=AttentionWindow.causal(), flags=capi.ATTENTION_BLOCKS)
    assert launched(backend) == (ROWS, cluster, 0)
    within(got, *ref.attention(q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, rolling=layout == "rolling"))
    assert not got[1].any()


@pytest.mark.parametrize("kdt,vdt", ALL, ids=IDS)
@pytest.mark.parametrize("L,Hq,H,D", [(9, 28, 4, 64), (130, 4, 4, 64), (33, 8, 4, 128), (50, 6, 2, 256)])
@pytest.mark.parametrize("layout,page", [("plain", 0), ("paged", 24), ("rolling", 0)])
@pytest.mark.parametrize("cap", [0.0, 25.0])
def test_rows_with_windows_and_caps(sess, backend, L, Hq, H, D, layout, page, kdt, vdt, cap):
    B, T = 2, 300
    q, k, v = inputs([L, D, kdt], B, T, H, D, L, Hq, kdt, vdt)
    lens = [711, 300] if layout == "rolling" else [300, 137]
    pos = causal(lens, L)
    got, _ = run_attention(sess, q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, layout=layout, page=page,
                           window=AttentionWindow(left=150, right=0), cap=cap, flags=capi.ATTENTION_BLOCKS)
    assert launched(backend)[0] == ROWS
    within(got, *ref.attention(q, k, v, kdt, vdt, scale=D ** -0.5, positions=pos, lengths=lens, rolling=layout == "rolling", left=150, cap=cap))


@pytest.mark.parametrize("T,L,first", [(1, 1, 7), (3, 2, 50), (5, 9, 2), (16, 4, 100), (17, 4, 2**31 - 21)])
@pytest.mark.parametrize("flags,kernel", [(capi.ATTENTION_ROW_UNITS, BOXES), (capi.ATTENTION_BLOCKS, ROWS)], ids=["columns", "rows"])
def test_tiny_rings_and_late_steps_in_boxes(sess, backend, T, L, first, flags, kernel):
    B, H, D = 1, 4, 64
    q, k, v = inputs([T, L], B, T, H, D, L, 8, Q8, Q4)
    pos = first + np.arange(L, dtype=np.int64)[None]
    lens = [int(pos[0, -1]) + 1]
    got, _ = run_attention(sess, q, k, v, Q8, Q4, scale=0.1, positions=pos.astype(np.int32), lengths=lens, layout="rolling",
                           window=AttentionWindow.causal(), flags=flags)
    assert launched(backend)[0] == (kernel if L > 1 else BOXES)
    within(got, *ref.attention(q, k, v, Q8, Q4, scale=0.1, positions=pos, lengths=lens, rolling=True))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("D,H,vdt", [(64, 4, Q8), (128, 2, Q4), (256, 1, Q8)])
@pytest.mark.parametrize("T,cluster", [(90, 1), (1100, 4)])
@pytest.mark.parametrize("flags,kernel", [(capi.ATTENTION_ROW_UNITS, BOXES), (capi.ATTENTION_BLOCKS, ROWS)], ids=["columns", "rows"])
def test_v_scales_that_are_not_finite_spoil_their_own_block(sess, backend, bad, D, H, vdt, T, cluster, flags, kernel):
    """One V scale of NaN or an infinity, in the last block of the last head: the rows that see its key have no finite value in the
    block's 32 dimensions and their true values elsewhere; rows that do not see it, and other heads, are clean."""
    B, L, Hq, at = 1, 12, 2 * H, T - 15
    q, k, v = inputs([5], B, T, H, D, L, Hq, Q8, vdt)
    pos = np.arange(T - 20, T - 20 + L, dtype=np.int32)[None]
    kw = dict(scale=0.1, positions=pos, lengths=[T])
    want, bound = ref.attention(q, k, v, Q8, vdt, **kw)
    v.reshape(B, T, H, D // 32, -1)[0, at, -1, -1, :2] = np.frombuffer(np.float16(bad).tobytes(), np.uint8)
    got, _ = run_attention(sess, q, k, v, Q8, vdt, window=AttentionWindow.causal(), flags=flags, **kw)
    assert launched(backend)[0] == kernel
    if kernel == ROWS:
        assert launched(backend)[1] == cluster
    clean = np.ones(got.shape, bool)
    clean[:, 5:, Hq - Hq // H:, D - 32:] = False
    assert not np.isfinite(got[~clean]).any()
    assert (np.abs(got - want)[clean] <= bound[clean]).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, 65504.0])
@pytest.mark.parametrize("D,H", [(64, 4), (128, 2), (256, 1)])
@pytest.mark.parametrize("flags,kernel", [(capi.ATTENTION_ROW_UNITS, BOXES), (capi.ATTENTION_BLOCKS, ROWS)], ids=["columns", "rows"])
def test_key_rows_that_only_later_rows_see(sess, backend, bad, D, H, flags, kernel):
    """A key row of NaN, infinite or huge scales: the rows before it (causal) are those of a clean cache."""
    B, T, L = 1, 90, 12
    q, k, v = inputs([3], B, T, H, D, L, 8 * H, Q8, Q8)
    pos = np.arange(70, 70 + L, dtype=np.int32)[None]
    want, bound = ref.attention(q, k, v, Q8, Q8, scale=0.1, positions=pos, lengths=[T])
    k.reshape(B, T, H, D // 32, 34)[0, 76, :, :, :2] = np.frombuffer(np.float16(bad).tobytes(), np.uint8)
    got, _ = run_attention(sess_quiet(sess), q, k, v, Q8, Q8, scale=0.1, positions=pos, lengths=[T], window=AttentionWindow.causal(), flags=flags)
    assert launched(backend)[0] == kernel
    within(got[:, :6], want[:, :6], bound[:, :6])


@pytest.mark.parametrize("D,H,kernel", [(64, 1, COLUMNS), (128, 1, COLUMNS), (256, 1, BOXES)])
@pytest.mark.parametrize("L", [1, 2])
def test_a_single_unit_with_more_keys_than_a_cluster_walks(sess, backend, D, H, kernel, L):
    """Dealt clusters: their sums meet in global memory, and the last of them to arrive adds them up, the same way every time."""
    T = 6000
    q, k, v = inputs([D, L], 1, T, H, D, L, 4, Q8, Q4)
    pos = causal([T], L)
    kw = dict(scale=D ** -0.5, positions=pos, lengths=[T], window=AttentionWindow.causal(), flags=capi.ATTENTION_ROW_UNITS)
    got, step = run_attention(sess, q, k, v, Q8, Q4, **kw)
    assert launched(backend) == (kernel, 8, 1)
    within(got, *ref.attention(q, k, v, Q8, Q4, scale=D ** -0.5, positions=pos, lengths=[T]))
    for _ in range(3):
        sess[1].write(step.out, np.zeros(q.shape, np.float32))
        sess[0].execute([step])
        assert np.array_equal(sess[1].read(step.out), got)


@pytest.mark.parametrize("kdt,vdt", [(Q8, Q4), (Q4, Q8)])
@pytest.mark.parametrize("H,kernel", [(4, BOXES), (3, COLUMNS)])
@pytest.mark.parametrize("layout,page", [("plain", 0), ("paged", 1000)])
def test_long_uneven_requests_are_dealt_by_their_keys(sess, backend, kdt, vdt, H, kernel, layout, page):
    """Many tiles for each warp, and requests from none to all of the context."""
    B, D, L, T = 8, 64, 1, 24000 if H == 4 else 32000
    lens = [T, 0, 1, T // 2, 16, T - 1, T // 3, 5000]
    q, k, v = inputs([H, kdt], B, T, H, D, L, 2 * H, kdt, vdt)
    pos = causal(lens, L)
    got, _ = run_attention(sess, q, k, v, kdt, vdt, scale=0.125, positions=pos, lengths=lens, layout=layout, page=page, window=AttentionWindow.causal())
    ran = launched(backend)
    assert ran[0] == kernel and ran[2] == 1
    within(got, *ref.attention(q, k, v, kdt, vdt, scale=0.125, positions=pos, lengths=lens))
    assert not got[1].any()


def test_the_forced_kernels_that_operands_allow(sess, backend):
    """Which kernel runs: ATTENTION_BLOCKS holds where rows are whole 16 bytes and more than one position is asked for, else columns do
    the work; other head sizes are any-shape."""
    for L, D, H, flags, kernel in ((2, 128, 2, capi.ATTENTION_BLOCKS, ROWS), (2, 128, 1, capi.ATTENTION_BLOCKS, COLUMNS), (1, 128, 2, capi.ATTENTION_BLOCKS, BOXES),
                                   (2, 128, 2, capi.ATTENTION_ROW_UNITS, BOXES), (2, 128, 2, capi.ATTENTION_GENERIC, ANY), (2, 96, 2, capi.ATTENTION_BLOCKS, ANY)):
        q, k, v = inputs([L, D], 1, 50, H, D, L, 4, Q8, Q8)
        got, _ = run_attention(sess, q, k, v, Q8, Q8, scale=0.1, flags=flags)
        assert launched(backend)[0] == kernel, (L, D, H, flags)
        within(got, *ref.attention(q, k, v, Q8, Q8, scale=0.1, positions=np.zeros((1, L), int), lengths=[50], right=capi.WINDOW_UNBOUNDED))


# ---- precision: inputs whose f32 evaluation is exact but for a few known roundings --------------------------------------------
KERNELS = [("columns", capi.ATTENTION_ROW_UNITS, BOXES), ("rows", capi.ATTENTION_BLOCKS, ROWS)]
FORCED = dict(argvalues=[(f, k) for _, f, k in KERNELS], ids=[n for n, _, _ in KERNELS])


def blocks(dtype, codes, scales):
    """Stored rows from whole-number codes [..., D] and f16 scales [..., D / 32]."""
    codes = np.asarray(codes).reshape(*np.shape(codes)[:-1], -1, 32)
    head = np.asarray(scales, np.float16)[..., None].view(np.uint8)
    if dtype == Q8:
        body = codes.astype(np.int8).view(np.uint8)
    else:
        n = (codes + 8).astype(np.uint8)
        body = n[..., 0::2] | n[..., 1::2] << 4
    return np.concatenate([np.broadcast_to(head, (*body.shape[:-1], 2)), body], -1).reshape(*codes.shape[:-2], -1)


@pytest.mark.parametrize("flags,kernel", **FORCED)
@pytest.mark.parametrize("D,H", [(64, 4), (128, 2), (256, 1)])
@pytest.mark.parametrize("kdt", [Q8, Q4], ids=["q8", "q4"])
def test_logits_keep_the_low_bits_of_the_queries(sess, backend, kdt, D, H, flags, kernel):
    """q = (1 + 2^-18, 1) and keys (7, -7) S and (-7, 7) S in two dimensions of a block, S = 2^12: every product is exact in f32 and so is
    their sum, +-7 * 2^-6, so the weights' quotient is known. Beyond two roundings of the logit's move to base 2 only exp2 (2^-22),
    the weights' two f16 terms (2^-23) and the sums and the quotient of two weights (4 * 2^-24) round: below 2^-20 of values of size one."""
    L, T = 2, 32
    q = np.zeros((1, L, H, D), np.float32)
    q[..., 33], q[..., 50] = 1 + 2.0 ** -18, 1.0
    codes = np.zeros((1, T, H, D))
    codes[0, 0::2, :, 33], codes[0, 0::2, :, 50] = 7, -7
    codes[0, 1::2, :, 33], codes[0, 1::2, :, 50] = -7, 7
    k = blocks(kdt, codes, np.full((1, T, H, D // 32), 2.0 ** 12))
    sign = np.where(np.arange(T) % 2 == 0, 1, -1)[None, :, None, None]
    v = blocks(Q8, np.broadcast_to(sign * 64, codes.shape), np.full((1, T, H, D // 32), 1 / 64))
    got, _ = run_attention(sess, q, k, v, kdt, Q8, scale=1.0, flags=flags)
    assert launched(backend)[0] == kernel
    want = np.tanh(7 * 2.0 ** 12 * 2.0 ** -18)
    assert np.abs(got - want).max() <= 2.0 ** -20


@pytest.mark.parametrize("flags,kernel", **FORCED)
@pytest.mark.parametrize("vscale", [2.0 ** -13, 1.0, 2.0 ** 13])
def test_weights_are_exact_to_the_last_bits_whatever_the_values_size(sess, backend, vscale, flags, kernel):
    """Two keys, one with V = 0: out / v = w / (1 + w) with w = exp(-x), x in [0, 1/2). In f32: x to base 2 rounds three times
    (2^-24 x each), the difference once, exp2 is good to 2^-22, the weights' two f16 terms to 2^-23, sum, quotient and product round
    once each. As independent errors, uniform over these bounds, their root mean square is below
    sqrt(3 * 0.5^2 + 1 + 16 + 4 + 3) / sqrt(3) * 2^-24 = 2.9 * 2^-24, times 1 / (1 + w) <= 0.63."""
    L, H, D, Hq = 256, 2, 128, 2
    rng = np.random.default_rng(17)
    x = rng.integers(1, 2 ** 10, (1, L, Hq)).astype(np.float32) * 2.0 ** -11
    q = np.zeros((1, L, Hq, D), np.float32)
    q[..., 5] = x
    codes = np.zeros((1, 2, H, D))
    codes[0, 1, :, 5] = -1
    k = blocks(Q8, codes, np.ones((1, 2, H, D // 32)))
    vc = np.zeros((1, 2, H, D))
    vc[0, 1] = 64
    v = blocks(Q8, vc, np.full((1, 2, H, D // 32), vscale))
    got, _ = run_attention(sess, q, k, v, Q8, Q8, scale=1.0, flags=flags)
    assert launched(backend)[0] == kernel
    w = np.exp(-x.astype(np.float64))[..., None]
    rel = got / (64 * vscale) / (w / (1 + w)) - 1
    assert np.sqrt((rel[..., 0] ** 2).mean()) <= 0.63 * 2.9 * 2.0 ** -24


def spread_case(rng, kdt, vdt, T, L, H, D, Hq):
    """Queries of one dimension, keys that are whole numbers there: a logit is one exact product, in [-1, 1]."""
    q = np.zeros((1, L, Hq, D), np.float32)
    q[..., 5] = 2.0 ** -3
    codes = np.zeros((1, T, H, D))
    codes[..., 5] = rng.integers(-7, 8, (1, T, H))
    vc = rng.integers(-7, 8, (1, T, H, D))
    return q, codes, vc


def spread_bound(w, values, ymax):
    """The weights' errors (the logit's move to base 2 and the difference: 5 * 2^-24 of the largest logit, exp2 2^-22, two f16 terms
    2^-22) count twice (sum and quotient), sums of N terms N + 16 roundings, each of them times sum w |v| / sum w."""
    mean_abs = w @ np.abs(values) / w.sum()
    return (2 * (5 * ymax * 2.0 ** -24 + 2.0 ** -21) + (len(w) + 16) * 2.0 ** -24) * mean_abs


@pytest.mark.parametrize("flags,kernel", **FORCED)
@pytest.mark.parametrize("vdt", [Q8, Q4], ids=["q8", "q4"])
@pytest.mark.parametrize("D,H", [(64, 4), (128, 2), (256, 1)])
@pytest.mark.parametrize("small", [2.0 ** -4, 2.0 ** -9, 2.0 ** -14])
@pytest.mark.parametrize("seen", [False, True])
def test_a_huge_value_row_costs_the_others_nothing(sess, backend, D, H, vdt, small, seen, flags, kernel):
    """One key's V has scales of 65504, the others' are `small`: rows that do not see the key (causal), and rows that give it a weight
    of e^-100, keep f32's precision in what they make of the others."""
    L, T, at = 12, 60, 45
    rng = np.random.default_rng([D, vdt])
    q, codes, vc = spread_case(rng, Q8, vdt, T, L, H, D, 2 * H)
    if seen:
        q[..., 6], codes[0, at, :, 6] = 2.0 ** -3, -100
        codes[0, at, :, 5] = 0
        q[..., 6] *= 8.0
    pos = np.arange(at - 6, at - 6 + L, dtype=np.int32)[None] if not seen else np.full((1, L), T - 1, np.int32)
    k = blocks(Q8, codes, np.ones((1, T, H, D // 32)))
    vs = np.full((1, T, H, D // 32), small) * (1 + rng.integers(0, 512, (1, T, H, D // 32)) / 1024)
    vs[0, at] = 65504
    vs = vs.astype(np.float16)
    v = blocks(vdt, vc, vs)
    got, _ = run_attention(sess, q, k, v, Q8, vdt, scale=1.0, positions=pos, lengths=[T], window=AttentionWindow.causal(), flags=flags, spoil_rows=False)
    assert launched(backend)[0] == kernel
    vals = ref.unpack(vdt, v)
    for l in range(L):
        n = int(pos[0, l]) + 1
        if not seen and n > at:
            continue
        for h in range(2 * H):
            y = codes[0, :n, h // 2] @ q[0, l, h].astype(np.float64)
            w = np.exp(y - y.max())
            want, bound = w @ vals[0, :n, h // 2] / w.sum(), spread_bound(w, vals[0, :n, h // 2], 1.0)
            assert (np.abs(got[0, l, h] - want) <= bound).all(), (l, h, np.abs(got[0, l, h] - want).max(), bound.max())


@pytest.mark.parametrize("flags,kernel", **FORCED)
@pytest.mark.parametrize("vdt", [Q8, Q4], ids=["q8", "q4"])
@pytest.mark.parametrize("D,H", [(64, 4), (128, 2), (256, 1)])
@pytest.mark.parametrize("ratio", [2.0 ** 8, 2.0 ** 16, 2.0 ** 24])
def test_a_huge_block_costs_the_others_of_its_rows_little(sess, backend, D, H, vdt, ratio, flags, kernel):
    """The scales of one block of every V row are `ratio` times the others': these keep f32's precision. The rows kernel holds a value as
    two f16 terms of which the row's largest scale is at most 2^15 of 128 codes: half of f16's last bit, 2^-25, is 2^-32 of that scale."""
    L, T = 3, 50
    rng = np.random.default_rng([D, vdt, 1])
    q, codes, vc = spread_case(rng, Q8, vdt, T, L, H, D, 2 * H)
    if vdt == Q8:
        vc = rng.integers(-127, 128, vc.shape)
    k = blocks(Q8, codes, np.ones((1, T, H, D // 32)))
    vs = 2.0 ** -10 * (1 + rng.integers(0, 512, (1, T, H, D // 32)) / 1024)
    vs[..., -1] *= ratio
    v = blocks(vdt, vc, vs)
    got, _ = run_attention(sess, q, k, v, Q8, vdt, scale=1.0, flags=flags)
    assert launched(backend)[0] == kernel
    vals = ref.unpack(vdt, v)
    for l in range(L):
        for h in range(2 * H):
            y = codes[0, :, h // 2] @ q[0, l, h].astype(np.float64)
            w = np.exp(y - y.max())
            want, bound = w @ vals[0, :, h // 2] / w.sum(), spread_bound(w, vals[0, :, h // 2], 1.0)
            if kernel == ROWS:
                bound = bound + 2.0 ** -32 * vs[0, :, h // 2].max()
            assert (np.abs(got[0, l, h] - want) <= bound).all(), (l, h, np.abs(got[0, l, h] - want).max(), bound.max())


@pytest.mark.parametrize("L", [1, 3])
def test_pages_of_more_than_a_million_tokens(sess, backend, L):
    """A page may hold any number of tokens: two requests, each in a page of its own."""
    import torch

    from aion_b200.backend import Chunk, StepAttention, TensorMeta
    s, store = sess
    D, H, page, T = 64, 4, 1_100_003, 700
    q, k, v = inputs([L], 2, T, H, D, L, 8, Q4, Q4)
    tids, pools = [], []
    for x in (k, v):
        pool = torch.zeros((2, page, x[0, 0].size), dtype=torch.uint8, device="cuda")
        for b in range(2):
            pool[1 - b, :T] = torch.from_numpy(x[b].reshape(T, -1)).cuda()
        tids.append(store.bind(TensorMeta(Q4, (2, page, H, D), quant_axis=3), Chunk(pool.data_ptr(), 0, pool.numel())))
        pools.append(pool)
    torch.cuda.synchronize()
    lens, pos = [T, 123], causal([T, 123], L)
    put = lambda a: store.add(TensorMeta(capi.DTYPE_I32, a.shape), a)
    tq, to = store.add(TensorMeta(capi.DTYPE_F32, q.shape), q), store.add(TensorMeta(capi.DTYPE_F32, q.shape))
    s.execute([StepAttention(out=to, q=tq, k=tids[0], v=tids[1], scale=0.125, query_positions=put(pos), kv_lengths=put(np.array(lens, np.int32)),
                             window=AttentionWindow.causal(), page_table=put(np.array([[1], [0]], np.int32)), flags=capi.ATTENTION_BLOCKS)])
    within(store.read(to), *ref.attention(q, k, v, Q4, Q4, scale=0.125, positions=pos, lengths=lens))
    assert launched(backend)[0] == (ROWS if L > 1 else BOXES)


@pytest.mark.parametrize("flags,kernel", [*[(f, k) for _, f, k in KERNELS], (capi.ATTENTION_GENERIC, ANY)], ids=["columns", "rows", "any"])
@pytest.mark.parametrize("cap", [1e-45, 1e-40, 1e-38, 1e30])
def test_soft_caps_near_the_ends_of_f32(sess, backend, cap, flags, kernel):
    """A cap that f32 holds as a subnormal number: all logits are zero beside any value of V, those of a query of zeros too. One far
    above the logits changes nothing."""
    T, H, D, L = 40, 2, 128, 3
    q, k, v = inputs([2], 1, T, H, D, L, 4, Q8, Q4)
    q[:, 0] = 0.0
    got, _ = run_attention(sess, q, k, v, Q8, Q4, scale=0.1, cap=cap, flags=flags)
    assert launched(backend)[0] == kernel
    kw = dict(positions=np.zeros((1, L), int), lengths=[T], right=capi.WINDOW_UNBOUNDED)
    want, bound = ref.attention(q, k, v, Q8, Q4, scale=0.1, **kw)
    if cap < 1:
        want, bound = ref.attention(0 * q, k, v, Q8, Q4, scale=0.1, **kw)
    else:
        # the division and the tanh of a small number: 2^-21 of a logit, which counts twice
        top = 0.1 * np.abs(np.einsum("lhd,thd->lht", q[0].astype(np.float64), np.repeat(ref.unpack(Q8, k)[0], 2, 1))).max()
        bound = bound + 2.0 ** -20 * top * np.abs(ref.unpack(Q4, v)).max()
    within(got, want, bound)
