"""Quantized-cache steps, what needs no GPU: struct layouts, refusals, and every cache row the kernels' index arithmetic names."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest

from aion_b200 import capi
from aion_b200.backend import (BackendError, Chunk, CudaSession, DeviceStore, StepAttention, StepQKNormRopeAppend, StepSequenceAppend,
                               StepSequenceRead, TensorMeta)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, Q4, Q8, I32 = capi.DTYPE_F32, capi.DTYPE_F16, capi.DTYPE_Q4_0, capi.DTYPE_Q8_0, capi.DTYPE_I32
OP = capi.Operand(1 << 20, 0, 1 << 40)   # never dereferenced: every call below is refused before any CUDA call


def test_struct_layouts(tmp_path):
    structs = {"AionCudaSequenceRead": capi.SequenceRead, "AionCudaQKNormRopeAppend": capi.QKNormRopeAppend,
               "AionCudaSequenceAppend": capi.SequenceAppend}
    text = open(os.path.join(ROOT, "include", "aion_cuda.h")).read()
    assert set(re.findall(r"^struct (\w+) \{", text, re.M)) == {"AionCudaSequenceRead", "AionCudaQKNormRopeAppend"}
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{os.path.join(ROOT, "include", "aion_cuda.h")}"', "int main(void) {"]
    for name, ct in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in ct._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-o", str(exe), str(src)], check=True)
    out = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, ct in structs.items():
        assert int(out[name]) == C.sizeof(ct)
        for f, _ in ct._fields_:
            assert int(out[f"{name}.{f}"]) == getattr(ct, f).offset, (name, f)


# ---- refusals of the C entry points --------------------------------------------------------
_fake = C.create_string_buffer(1 << 16)   # stands in for a device object that is never reached


def _call(fn, rec):
    return getattr(capi.load(), fn)(C.cast(_fake, C.c_void_p), C.byref(rec)), capi.last_error()


def _append(**kw):
    a = dict(cache=OP, new_kv=OP, end_index=OP, batch=2, t_cap=64, heads=2, head_dim=64, new_len=1, dtype=Q8, new_dtype=F32)
    a.update(kw)
    return capi.SequenceAppend(**a)


def _read(**kw):
    a = dict(out=OP, cache=OP, batch=2, t_cap=64, heads=2, head_dim=64, out_len=3, dtype=Q8, out_dtype=F32)
    a.update(kw)
    return capi.SequenceRead(**a)


def _rope(**kw):
    a = dict(q_out=OP, qkv=OP, q_gamma=OP, k_gamma=OP, positions=OP, end_index=OP, k_cache=OP, v_cache=OP, batch=2, len=1, h_q=4, h_kv=2,
             head_dim=64, t_cap=64, eps=1e-6, base_frequency=1e4, scale_factor=1.0, proportion=1.0, k_dtype=Q8, v_dtype=Q4)
    a.update(kw)
    return capi.QKNormRopeAppend(**a)


def _attn(**kw):
    a = dict(out=OP, q=OP, k=OP, v=OP, q_dtype=F32, k_dtype=Q8, v_dtype=Q8, batch=2, l_q=1, h_q=4, h_kv=2, d_k=64, d_v=64, t_cap=64, scale=1.0)
    a.update(kw)
    return capi.Attention(**a)


INV, UNS = capi.INVALID_ARGUMENT, capi.UNSUPPORTED


@pytest.mark.parametrize("fn,rec,status", [
    ("aion_cuda_sequence_append", _append(new_dtype=Q8), INV),
    ("aion_cuda_sequence_append", _append(head_dim=48), UNS),
    ("aion_cuda_sequence_append", _append(t_cap=0), INV),
    ("aion_cuda_sequence_append", _append(t_cap=1 << 32), UNS),
    ("aion_cuda_sequence_append", _append(page_table=OP, page_tokens=0, pool_pages=4), INV),
    ("aion_cuda_sequence_append", _append(page_table=OP, page_tokens=16, pool_pages=0), INV),
    ("aion_cuda_sequence_append", _append(page_table=OP, page_tokens=16, pool_pages=4, rolling=1), UNS),
    ("aion_cuda_sequence_append", _append(batch=1 << 20, new_len=1 << 20), UNS),
    ("aion_cuda_sequence_read", _read(dtype=I32), INV),
    ("aion_cuda_sequence_read", _read(out_dtype=Q8), INV),
    ("aion_cuda_sequence_read", _read(head_dim=80), UNS),
    ("aion_cuda_sequence_read", _read(t_cap=0), INV),
    ("aion_cuda_sequence_read", _read(page_table=OP, page_tokens=16, pool_pages=4, rolling=1), UNS),
    ("aion_cuda_qk_norm_rope_append", _rope(k_dtype=F32), INV),
    ("aion_cuda_qk_norm_rope_append", _rope(v_dtype=I32), INV),
    ("aion_cuda_qk_norm_rope_append", _rope(eps=0.0), INV),
    ("aion_cuda_qk_norm_rope_append", _rope(eps=float("nan")), INV),
    ("aion_cuda_qk_norm_rope_append", _rope(head_dim=63), INV),
    ("aion_cuda_qk_norm_rope_append", _rope(head_dim=2048), INV),
    ("aion_cuda_qk_norm_rope_append", _rope(head_dim=40), UNS),
    ("aion_cuda_qk_norm_rope_append", _rope(ld_qkv=100), INV),
    ("aion_cuda_qk_norm_rope_append", _rope(proportion=float("nan")), INV),
    ("aion_cuda_qk_norm_rope_append", _rope(t_cap=0), INV),
    ("aion_cuda_qk_norm_rope_append", _rope(batch=1 << 20, len=1 << 20), UNS),
    ("aion_cuda_attention", _attn(q_dtype=Q8), INV),
    ("aion_cuda_attention", _attn(k_dtype=I32), INV),
    ("aion_cuda_attention", _attn(t_cap=0), INV),
    ("aion_cuda_attention", _attn(scale=0.0), INV),
])
def test_refusals(fn, rec, status):
    got, message = _call(fn, rec)
    assert got == status, (got, message)
    assert fn.removeprefix("aion_cuda_") in message


@pytest.mark.parametrize("fn,rec", [("aion_cuda_sequence_append", _append(batch=0)), ("aion_cuda_sequence_append", _append(new_len=0)),
                                    ("aion_cuda_sequence_read", _read(out_len=0)), ("aion_cuda_qk_norm_rope_append", _rope(len=0))])
def test_empty_steps_do_nothing(fn, rec):
    assert _call(fn, rec)[0] == capi.OK


def test_null_records():
    lib = capi.load()
    for fn in ("aion_cuda_sequence_append", "aion_cuda_sequence_read", "aion_cuda_qk_norm_rope_append", "aion_cuda_attention"):
        assert getattr(lib, fn)(None, None) == INV


# ---- refusals of the session ---------------------------------------------------------------
class _Backend:
    class device_memory:
        @staticmethod
        def alloc(*a):
            return 4096

    class _lib:
        def __getattr__(self, name):
            raise AssertionError("a refused step reached the library")

    _h = None


def _session(**metas):
    store = DeviceStore(_Backend.device_memory)
    backend = _Backend()
    backend._lib = _Backend._lib()
    return CudaSession(backend, store), {k: store.bind(m, Chunk(4096, 0, m.nbytes())) for k, m in metas.items()}


def _cache(dtype=Q8, shape=(2, 64, 2, 64), axis=3, policy="none"):
    return TensorMeta(dtype, shape, quant_axis=axis, cache_policy=policy)


@pytest.mark.parametrize("cache,new,index", [
    (_cache(axis=0), TensorMeta(F32, (2, 1, 2, 64)), TensorMeta(I32, (2,))),                    # quantized along the wrong axis
    (_cache(policy="growable"), TensorMeta(F32, (2, 1, 2, 64)), TensorMeta(I32, (2,))),
    (_cache(), TensorMeta(F32, (2, 1, 2, 32)), TensorMeta(I32, (2,))),
    (_cache(), TensorMeta(F32, (3, 1, 2, 64)), TensorMeta(I32, (3,))),
    (_cache(dtype=F16), TensorMeta(F32, (2, 1, 2, 64)), TensorMeta(I32, (2,))),                 # an f16 cache takes f16 rows
])
def test_session_refuses_an_append(cache, new, index):
    s, t = _session(cache=cache, new=new, index=index)
    with pytest.raises(BackendError):
        s.execute([StepSequenceAppend(cache=t["cache"], new_kv=t["new"], end_index=t["index"])])


def test_session_refuses_reads_and_fused_appends():
    s, t = _session(cache=_cache(), bad_axis=_cache(axis=1), out=TensorMeta(F32, (2, 5, 2, 64)), wide=TensorMeta(F32, (2, 5, 3, 64)),
                    index=TensorMeta(I32, (2,)), index3=TensorMeta(I32, (3,)), table=TensorMeta(I32, (3, 4)), q=TensorMeta(F32, (2, 1, 4, 64)),
                    qkv=TensorMeta(F32, (2, 1, 8 * 64)), short=TensorMeta(F32, (2, 1, 7 * 64)), pos=TensorMeta(I32, (2, 1)),
                    gamma=TensorMeta(F32, (64,)), gamma32=TensorMeta(F32, (32,)), half=TensorMeta(F16, (2, 64, 2, 32)), ring=_cache(policy="rolling"))
    read = lambda **kw: StepSequenceRead(**{**dict(out=t["out"], cache=t["cache"]), **kw})
    rope = lambda **kw: StepQKNormRopeAppend(**{**dict(q_out=t["q"], qkv=t["qkv"], positions=t["pos"], end_index=t["index"], k_cache=t["cache"],
                                                       v_cache=t["cache"], base_frequency=1e4, q_gamma=t["gamma"]), **kw})
    attn = lambda **kw: StepAttention(**{**dict(out=t["q"], q=t["q"], k=t["cache"], v=t["cache"]), **kw})
    for step in (read(cache=t["bad_axis"]), read(out=t["wide"]), read(start_index=t["index3"]), read(lengths=t["gamma"]), read(page_table=t["table"]),
                 rope(k_cache=t["bad_axis"]), rope(qkv=t["short"]), rope(q_gamma=t["gamma32"]), rope(end_index=t["index3"]), rope(v_cache=t["half"]), rope(v_cache=t["ring"]), rope(k_cache=t["ring"]),
                 rope(positions=t["index"]), attn(k=t["bad_axis"]), attn(v=t["bad_axis"])):
        with pytest.raises(BackendError):
            s.execute([step])


# ---- the rows that the index arithmetic names -------------------------------------------------
PROGRAM = r"""
#include <cstdio>
#include "%s/aion_b200/csrc/cache_geom.cuh"
using namespace aion;
int main() {
  // stdin: t_cap page pages_per_request pool rolling batch new_len, the table, then end_index, start and length of each request
  unsigned t_cap, page, per, pool, rolling, batch, n;
  while (scanf("%%u %%u %%u %%u %%u %%u %%u", &t_cap, &page, &per, &pool, &rolling, &batch, &n) == 7) {
    static int32_t table[4096], e[64], s[64], len[64];
    for (unsigned i = 0; i < batch * per; i++) scanf("%%d", table + i);
    for (unsigned i = 0; i < batch; i++) scanf("%%d %%d %%d", e + i, s + i, len + i);
    CacheGeom g{page ? table : nullptr, t_cap, page, per, pool, rolling};
    for (unsigned b = 0; b < batch; b++) {
      for (unsigned t = 0; t < n; t++) {
        bool bad;
        long long r = append_row(g, b, e[b], t, n, &bad);
        printf("%%lld %%d ", r, (int)bad);
      }
      ReadSpan sp = read_span(g, s, len, b);
      printf("%%u %%u %%d\n", sp.lo, sp.hi, (int)sp.bad);
    }
  }
}
"""


def _expected(t_cap, page, table, pool, rolling, e, s, length, n):
    """What the arithmetic has to say, request by request, from the definition."""
    lines = []
    for b in range(len(e)):
        row = []
        fits = e[b] >= 0 and (rolling or e[b] + n <= t_cap)
        for t in range(n):
            if not fits:
                row += [-1, 1]
            elif rolling:
                row += [-1 if any((e[b] + u) % t_cap == (e[b] + t) % t_cap for u in range(t + 1, n)) else b * t_cap + (e[b] + t) % t_cap, 0]
            elif page:
                pg = table[b][(e[b] + t) // page]
                ok = 0 <= pg < pool
                row += [pg * page + (e[b] + t) % page if ok else -1, 0 if ok else 1]
            else:
                row += [b * t_cap + e[b] + t, 0]
        bad = s[b] < 0 or length[b] < 0 or (not rolling and length[b] > t_cap)
        row += [0, 0, 1] if bad else [max(0, length[b] - t_cap) if rolling else 0, length[b], 0]
        lines.append(row)
    return lines


def test_every_row_the_kernels_name_is_the_right_one(tmp_path):
    src = tmp_path / "geom.cpp"
    src.write_text(PROGRAM % ROOT)
    exe = tmp_path / "geom"
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined,address", "-o", str(exe), str(src)], check=True)
    rng = np.random.default_rng(3)
    text, want = [], []
    for trial in range(200):
        t_cap, batch, n = int(rng.integers(1, 60)), int(rng.integers(1, 5)), int(rng.integers(1, 70))
        kind = trial % 3   # contiguous, ring, paged
        page = int(rng.integers(1, 20)) if kind == 2 else 0
        per = -(-t_cap // page) if page else 0
        pool = batch * per + 1 if page else 0
        table = rng.permutation(max(1, batch * per + 1))[: batch * per].reshape(batch, per) if page else np.zeros((batch, 0), int)
        if page and trial % 4 == 2:   # page numbers outside the pool
            table[rng.integers(batch), rng.integers(per)] = rng.choice([-1, -2**31, pool, pool + 5, 2**31 - 1])
        e = [int(x) for x in rng.integers(-2, t_cap + 3, batch)]
        if kind == 1:
            e = [int(x) for x in rng.choice([0, 1, t_cap - 1, 5 * t_cap + 3, 2**31 - 1], batch)]
        s = [int(x) for x in rng.integers(-1, t_cap, batch)]
        length = [int(x) for x in rng.integers(-1, t_cap + 2, batch)] if kind != 1 else [int(x) for x in rng.choice([0, 1, t_cap, t_cap + 7, 2**31 - 1], batch)]
        text.append(f"{t_cap} {page} {per} {pool} {int(kind == 1)} {batch} {n} " + " ".join(str(int(x)) for x in table.reshape(-1)) + " " +
                    " ".join(f"{e[b]} {s[b]} {length[b]}" for b in range(batch)))
        want += _expected(t_cap, page, table.tolist(), pool, kind == 1, e, s, length, n)
    got = subprocess.run([str(exe)], input="\n".join(text), capture_output=True, text=True, check=True).stdout.splitlines()
    assert [[int(x) for x in line.split()] for line in got] == want


TILES = r"""
#include <cstdio>
#include "%s/aion_b200/csrc/cache_geom.cuh"
using namespace aion;
int main() {
  // stdin: t_cap page rolling lo hi; out: segment, first row in it and rows of every tile that holds keys [lo, hi)
  unsigned t_cap, page, rolling, lo, hi;
  while (scanf("%%u %%u %%u %%u %%u", &t_cap, &page, &rolling, &lo, &hi) == 5) {
    static int32_t table[1];
    const TileSpace ts = tile_space(CacheGeom{page ? table : nullptr, t_cap, page, page ? (t_cap + page - 1) / page : 0, 1, rolling});
    const TileRange r = tiles_of_keys(ts, lo, hi);
    for (unsigned tile = r.first; tile < r.end; tile++) {
      const unsigned seg = tile / ts.per_seg, in_seg = tile - seg * ts.per_seg;
      printf("%%u %%u %%u ", seg, in_seg * TILE_KEYS, tile_rows(ts, in_seg));
    }
    printf("\n");
  }
}
"""


def test_no_tile_of_attention_reaches_beyond_its_page_ring_or_cache(tmp_path):
    """Every tile that the attention kernels copy lies within its segment's rows (a page, a lap of the ring, the request's rows of a
    contiguous cache, whatever its length), and the tiles of a range of keys hold each of them once, in order."""
    src = tmp_path / "tiles.cpp"
    src.write_text(TILES % ROOT)
    exe = tmp_path / "tiles"
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined,address", "-o", str(exe), str(src)], check=True)
    cases = []
    for t_cap in (1, 2, 15, 16, 17, 31, 33, 90, 96, 700):
        for page, rolling in ((0, 0), (0, 1), (1, 0), (5, 0), (16, 0), (40, 0), (2**31 - 1, 0)):
            seg_len = page or t_cap
            cases += [(t_cap, page, rolling, lo, hi, seg_len) for lo in (0, 1, t_cap // 2, t_cap - 1) for hi in (lo, lo + 1, t_cap)]
            if rolling:
                cases += [(t_cap, page, 1, 5 * t_cap + 3, 6 * t_cap + 3, t_cap), (t_cap, page, 1, 2**31 - 1 - t_cap, 2**31 - 1, t_cap)]
    text = "\n".join(" ".join(map(str, c[:5])) for c in cases)
    out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.split("\n")
    for (t_cap, page, rolling, lo, hi, seg_len), line in zip(cases, out):
        v = [int(x) for x in line.split()]
        keys = []
        for seg, first, rows in zip(v[::3], v[1::3], v[2::3]):
            assert 0 < rows <= 16 and first + rows <= seg_len, (t_cap, page, rolling, lo, hi, seg, first, rows)
            keys += range(seg * seg_len + first, seg * seg_len + first + rows)
        assert keys == sorted(set(keys)) and set(range(lo, hi)) <= set(keys), (t_cap, page, rolling, lo, hi)


# ---- operands that overlap ----------------------------------------------------------------------
def _apart(**kw):
    """Operands of their own, a gigabyte apart, but for those that `kw` places: name=(other's name, bytes into it)."""
    def place(names):
        at = {n: (i + 1) << 30 for i, n in enumerate(names)}
        for n, (other, off) in kw.items():
            at[n] = at[other] + off
        return {n: capi.Operand(at[n], 0, 1 << 29) for n in names}
    return place


@pytest.mark.parametrize("fn,make,names,case", [
    *[("aion_cuda_sequence_append", _append, ("cache", "new_kv", "end_index"), {n: ("cache", off)})
      for n, off in (("new_kv", 0), ("new_kv", 2 * 64 * 2 * 68 - 4), ("end_index", 8))],
    ("aion_cuda_sequence_append", _append, ("cache", "new_kv", "end_index"), {"cache": ("new_kv", 2 * 2 * 64 * 4 - 2)}),
    *[("aion_cuda_sequence_read", _read, ("out", "cache", "start_index", "lengths"), {n: ("out", 4)}) for n in ("start_index", "lengths")],
    ("aion_cuda_sequence_read", _read, ("out", "cache", "start_index", "lengths"), {"cache": ("out", 2 * 3 * 2 * 64 * 4 - 4)}),
    *[("aion_cuda_qk_norm_rope_append", _rope, ("q_out", "qkv", "q_gamma", "k_gamma", "positions", "end_index", "k_cache", "v_cache"), {a: (b, 0)})
      for a, b in (("k_cache", "qkv"), ("v_cache", "qkv"), ("k_cache", "q_out"), ("q_out", "v_cache"), ("q_out", "qkv"), ("v_cache", "k_cache"),
                   ("q_gamma", "q_out"), ("positions", "k_cache"), ("end_index", "v_cache"))],
])
def test_operands_that_overlap_are_refused_before_any_cuda_call(fn, make, names, case):
    got, message = _call(fn, make(**_apart(**case)(names)))
    assert got == INV and "overlap" in message, (got, message)


@pytest.mark.parametrize("kw", [dict(k_dtype=Q8), dict(v_dtype=Q4), dict(k_dtype=F16, v_dtype=Q8, qk_norm=True), dict(k_dtype=Q8, v_dtype=Q8, head_dim=48),
                                dict(k_dtype=F32, v_dtype=F32), dict(k_dtype=F32, v_dtype=F16)], ids=str)
def test_a_decoder_whose_caches_attention_cannot_read_is_refused_when_it_is_built(kw):
    from aion_b200.decoder import DecoderConfig, SyntheticDecoder
    with pytest.raises(BackendError) as e:
        SyntheticDecoder(_Backend(), DecoderConfig(layers=1, **kw), 1, None, None)
    assert e.value.name == "Unsupported"


@pytest.mark.parametrize("rec,status", [
    (_attn(batch=1 << 30, l_q=1 << 30, h_q=16, h_kv=16), UNS),                                        # 2^64 rows: no rows modulo 2^64
    (_attn(batch=274177, l_q=1, h_q=1 << 40, h_kv=1), UNS),
    (_attn(k_dtype=F16, v_dtype=F16, batch=1 << 29, t_cap=(1 << 31) - 1, h_q=1, h_kv=1, d_k=128, d_v=128), UNS),
    (_attn(batch=1 << 29, t_cap=(1 << 31) - 1, h_q=1, h_kv=1), UNS),
    (_attn(page_table=OP, page_tokens=1 << 20, pool_pages=(1 << 44) + 1), INV),                       # 2^64 + 2^20 rows
    (_attn(page_table=OP, page_tokens=0, pool_pages=2), INV),
    (_attn(page_table=OP, page_tokens=1 << 30, pool_pages=2), INV),
])
def test_attention_refuses_sizes_whose_products_wrap(rec, status):
    got, message = _call("aion_cuda_attention", rec)
    assert got == status and "attention" in message, (got, message)
