"""The paged cache's operators on the GPU against float64: head layouts, pages,
lengths around the tiles' and splits' edges, rows that see nothing, non-finite
values at masked and visible places, pages that do not exist, strides, streams
and captured graphs, and a few steps of them together.

Bounds: an output is off by at most half a step of its type and what the fp32
sums and the probabilities' own rounding to the type leave (paged64.World)."""
import ctypes as C

import numpy as np
import pytest

import paged64
from paged64 import Dev, World, near, ref_append, to16, wide

pytestmark = pytest.mark.gpu

HEADS = [(1, 1, 64), (4, 2, 64), (16, 8, 128), (8, 1, 64), (6, 2, 128), (5, 1, 128), (16, 2, 128), (3, 3, 256), (8, 2, 256), (40, 2, 64)]


def _check_attention(mdx, w, **k):
    out, lse = w.attention(mdx, **k)
    ref, rlse, slack, lslack = w.ref_attention(k.get("scale") or None)
    taking_part = np.concatenate([np.arange(w.T)[w.q_start[r]:w.q_start[r] + min(w.new[r], w.max_q)] for r in range(w.R)] + [np.zeros(0, int)])
    assert near(out[taking_part], ref[taking_part], slack[taking_part], w.dtype) <= 0
    fin = np.isfinite(rlse[taking_part])
    assert np.array_equal(lse[taking_part][~fin], rlse[taking_part].astype(np.float32)[~fin], equal_nan=True)
    assert np.all(np.abs(lse[taking_part][fin] - rlse[taking_part][fin]) <= lslack[taking_part][fin])
    return out, lse


# ---- attention -----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_attention_single_tokens(mdx, gpu, nq, nkv, hd, dtype):
    """One new row per request, caches around the edges of tiles, pages and splits."""
    rng = np.random.default_rng(nq * hd)
    kv = [1, 2, 15, 16, 17, 31, 32, 33, 63, 127, 128, 129, 255, 256, 257, 511, 700]
    _check_attention(mdx, World(rng, dtype, nq, nkv, hd, 16, [1] * len(kv), kv).upload(mdx))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("dtype,nq,nkv,hd", [("fp16", 4, 2, 128), ("bf16", 4, 4, 64), ("bf16", 4, 1, 256)])
def test_attention_chunks_and_pages(mdx, gpu, dtype, nq, nkv, hd, page):
    """Chunks of different lengths behind different caches, single tokens among them."""
    rng = np.random.default_rng(page + hd)
    new, kv = [1, 2, 5, 16, 17, 33, 40, 64, 65, 100, 1], [1, 2, 300, 16, 50, 33, 141, 64, 321, 229, 513]
    _check_attention(mdx, World(rng, dtype, nq, nkv, hd, page, new, kv).upload(mdx))


@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_attention_chunks_and_heads(mdx, gpu, nq, nkv, hd):
    rng = np.random.default_rng(nq + hd)
    new, kv = [37, 1, 3, 130], [90, 333, 3, 200]
    _check_attention(mdx, World(rng, "fp16", nq, nkv, hd, 32, new, kv).upload(mdx))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attention_of_one_long_chunk(mdx, gpu, dtype):
    rng = np.random.default_rng(5)
    _check_attention(mdx, World(rng, dtype, 4, 2, 128, 64, [515], [1203]).upload(mdx))
    _check_attention(mdx, World(rng, dtype, 2, 2, 64, 64, [400], [400]).upload(mdx))


@pytest.mark.parametrize("dtype,hd", [("fp16", 128), ("bf16", 64)])
def test_attention_over_a_long_cache(mdx, gpu, dtype, hd):
    """More splits than a wave has lanes, and a short cache beside it."""
    rng = np.random.default_rng(6)
    _check_attention(mdx, World(rng, dtype, 2, 1, hd, 64, [1, 1], [40003, 5]).upload(mdx))


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 33]])
def test_attention_rows_that_see_nothing(mdx, gpu, new):
    """More new rows than the cache has: the first see nothing and get zeros; an empty cache; a request without new rows."""
    rng = np.random.default_rng(7)
    w = World(rng, "fp16", 4, 2, 64, 16, new + [0, 5], [0, 1, max(new[2] - 3, 0), 20, 2]).upload(mdx)
    out, lse = _check_attention(mdx, w)
    assert not out[:new[0]].any() and np.all(lse[:new[0]] == -np.inf)


@pytest.mark.parametrize("new,kv", [([1], [33]), ([1, 1], [600, 40]), ([3, 64], [20, 100])])
def test_attention_leaves_out_what_a_batch_does_not_name(mdx, gpu, new, kv):
    """Rows behind the last request, gaps between strided rows, rows past max_q_len and cache rows past max_kv_len."""
    rng = np.random.default_rng(8)
    w = World(rng, "bf16", 4, 2, 64, 32, new, kv).upload(mdx)
    ref, rlse, slack, _ = w.ref_attention()
    T, width, gap = w.T + 3, 4 * 64, 4 * 64 + 24
    q = np.zeros((T, gap), np.uint16)
    q[:w.T, :width] = w.q.reshape(w.T, width)
    q[w.T:] = to16(np.full((3, gap), np.nan, np.float32), "bf16")
    dq, out, lse = Dev(mdx, q), Dev(mdx, np.full((T, gap + 8), 0x1234, np.uint16)), Dev(mdx, np.full((T, 4), 5.0, np.float32))
    b = mdx.paged_batch(w.R, T, w.max_q, w.max_kv, w.max_pages, w.d["q_start"], w.d["kv_len"], w.d["table"])
    need = mdx.paged_attention_workspace(w.cache, b)
    ws = Dev(mdx, np.full(need + 64, 0xab, np.uint8))
    mdx.paged_attention(w.cache, b, dq, out, ws, need, lse=lse, q_stride=gap, out_stride=gap + 8)
    o = out.get()
    assert near(o[:w.T, :width].reshape(ref.shape), ref, slack, "bf16") <= 0
    assert np.all(o[:, width:] == 0x1234) and np.all(o[w.T:] == 0x1234) and np.all(lse.get()[w.T:] == 5.0)
    assert np.all(ws.get()[need:] == 0xab)
    # the same with lengths that the batch cuts
    w2 = World(rng, "bf16", 4, 2, 64, 32, new, kv, max_q=2, max_kv=36).upload(mdx)
    _check_attention(mdx, w2)


def test_attention_shared_and_missing_pages(mdx, gpu):
    """Two requests over the same pages; pages that do not exist count as absent rows."""
    rng = np.random.default_rng(9)
    w = World(rng, "fp16", 4, 2, 128, 16, [1, 20, 1, 3, 1], [200, 120, 200, 64, 40])
    w.table[2] = w.table[0]
    w.table[1, 2], w.table[1, 7], w.table[3, 0] = -5, w.n_pages, 2 ** 31 - 1
    w.table[4, :] = -1                                  # none at all: sees nothing
    out, lse = _check_attention(mdx, w.upload(mdx))
    assert not out[-1].any() and np.all(lse[-1] == -np.inf)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_attention_missing_pages_beside_a_page_of_nan(mdx, gpu, page, hd):
    """Nothing of page 0 shows, which no request holds, where a chunk's pages do not exist (at the beginning, between others, at the end)."""
    rng = np.random.default_rng(17)
    w = World(rng, "fp16", 2, 1, hd, page, [70, 1, 130], [900, 700, 777])
    free = (set(range(w.n_pages)) - set(w.table[w.table >= 0])).pop()
    w.table[w.table == 0] = free
    w.k[0], w.v[0] = (to16(np.full(w.k[0].shape, np.nan, np.float32), "fp16") for _ in range(2))
    n = w.n_pages
    w.table[0, 0], w.table[0, 256 // page], w.table[1, 1], w.table[2, 512 // page], w.table[2, -(-777 // page) - 1] = -1, n, -7, n + 5, -1
    _check_attention(mdx, w.upload(mdx))


@pytest.mark.parametrize("dtype,hd", [("bf16", 64), ("fp16", 128), ("bf16", 256)])
@pytest.mark.parametrize("kv", [511, 512, 513, 640, 705, 1025])
def test_attention_ends_of_long_chunks(mdx, gpu, dtype, hd, kv):
    """Caches that end at, before and behind a tile, with several tiles on their way."""
    rng = np.random.default_rng(kv)
    _check_attention(mdx, World(rng, dtype, 4, 2, hd, 128, [33, kv - 300, 1], [kv, kv, 3]).upload(mdx))


BAD = {"nan": np.nan, "inf": np.inf, "-inf": -np.inf}


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("what", list(BAD))
@pytest.mark.parametrize("new,kv", [([1, 1], [20, 600]), ([4, 1], [100, 33]), ([70, 40], [150, 40])])
def test_attention_non_finite_rows_behind_the_last(mdx, gpu, new, kv, what, dtype):
    """K and V rows of the pool that no request holds."""
    rng = np.random.default_rng(10)
    w = World(rng, dtype, 4, 2, 64, 64, new, kv)
    held = np.zeros((w.n_pages, w.page), bool)
    for r in range(w.R):
        _, pg, slot, _ = w.where(r)
        held[pg, slot] = True
    bits = to16(np.float32(BAD[what]), dtype)
    for x in (w.k, w.v):
        x.transpose(0, 2, 1, 3)[~held] = bits
    _check_attention(mdx, w.upload(mdx))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("what", list(BAD))
@pytest.mark.parametrize("new,kv,row", [([1], [40], 17), ([1], [700], 300), ([6], [70], 67), ([100], [100], 50), ([100], [171], 120), ([1], [1], 0)])
def test_attention_non_finite_values(mdx, gpu, new, kv, row, what, which, dtype):
    """A value that some rows see and, in a chunk, others do not: those it does not reach stay finite."""
    rng = np.random.default_rng(11)
    w = World(rng, dtype, 4, 2, 64, 16, new, kv)
    pg, slot = w.table[0, row // 16], row % 16
    getattr(w, which)[pg, 1, slot, 13] = to16(np.float32(BAD[what]), dtype)
    w.q[:, :, 13] = to16(np.abs(wide(w.q[:, :, 13], dtype)) + 0.25, dtype)     # the sign of q . K is known
    _check_attention(mdx, w.upload(mdx))


@pytest.mark.parametrize("new,kv", [([1, 1], [40, 700]), ([40, 1], [60, 33])])
def test_attention_all_scores_minus_infinity(mdx, gpu, new, kv):
    """Keys that are all -inf are seen (NaN, as the arithmetic has it), which is not the same as seeing nothing."""
    rng = np.random.default_rng(12)
    w = World(rng, "fp16", 2, 1, 64, 32, new, kv)
    w.q = to16(np.abs(wide(w.q, "fp16")) + 0.25, "fp16")
    w.k[w.table[0][w.table[0] >= 0]] = to16(np.float32(-np.inf), "fp16")
    out, lse = _check_attention(mdx, w.upload(mdx))
    assert np.all(np.isnan(wide(out[0], "fp16"))) and np.all(np.isneginf(lse[0]))


@pytest.mark.parametrize("dtype,std,q_std", [("fp16", 200.0, 60.0), ("bf16", 1e15, 1e15), ("fp16", 1e-4, 1e-4), ("bf16", 1e-20, 1.0), ("fp16", 1.0, 20.0)])
@pytest.mark.parametrize("new,kv", [([1, 1], [40, 600]), ([50], [130])])
def test_attention_large_and_small_values(mdx, gpu, dtype, std, q_std, new, kv):
    """Scores far beyond the exponential's range, and values next to the types' ends."""
    rng = np.random.default_rng(13)
    w = World(rng, dtype, 2, 2, 64, 16, new, kv, std=std, q_std=q_std).upload(mdx)
    _check_attention(mdx, w)
    _check_attention(mdx, w, scale=0.03)


@pytest.mark.parametrize("dtype,nq,nkv,hd", [("fp16", 16, 8, 64), ("bf16", 24, 8, 128)])
def test_attention_chunks_beside_single_tokens(mdx, gpu, dtype, nq, nkv, hd):
    """More blocks than CUs: chunks and short requests go through kernels of their own, both with splits."""
    rng = np.random.default_rng(16)
    new = [1] * 44
    new[3], new[17], new[18], new[43] = 40, 17, 2, 33
    kv = [int(x) for x in rng.integers(1, 120, 44) + np.array(new)]
    kv[0], kv[3], kv[5] = 1100, 1300, 513
    _check_attention(mdx, World(rng, dtype, nq, nkv, hd, 32, new, kv).upload(mdx))


@pytest.mark.parametrize("requests", [64, 65, 150])
def test_attention_many_requests(mdx, gpu, requests):
    """More requests than a wave has lanes, empty ones among them."""
    rng = np.random.default_rng(requests)
    new = [int(x) for x in rng.choice([0, 1, 1, 1, 3, 40], requests)]
    new[0], new[-1] = 70, 41
    kv = [n + int(x) for n, x in zip(new, rng.integers(0, 60, requests))]
    w = World(rng, "fp16", 2, 1, 64, 16, new, kv).upload(mdx)
    _, lse = _check_attention(mdx, w)
    _check_mass(mdx, w, np.nan_to_num(lse, nan=0.0, neginf=-np.inf))


def test_attention_on_two_streams(mdx, gpu):
    """Calls at once, each with its own workspace and outputs, against the same ones alone."""
    H = _hip()
    rng = np.random.default_rng(17)
    worlds = [World(rng, "fp16", 8, 4, 128, 64, *x).upload(mdx) for x in (([1] * 8, [3000] * 8), ([300], [2000]), ([1, 60, 1], [700, 900, 20]))]
    alone = [w.attention(mdx) for w in worlds]
    streams = [C.c_void_p() for _ in worlds]
    outs = []
    for w, st in zip(worlds, streams):
        assert H.hipStreamCreate(C.byref(st)) == 0
        need = mdx.paged_attention_workspace(w.cache, w.batch)
        outs.append((Dev(mdx, np.zeros(w.q.shape, np.uint16)), Dev(mdx, np.zeros((w.T, w.nq), np.float32)), Dev(mdx, np.zeros(max(need, 16), np.uint8)), need))
    assert mdx.lib().mdx_device_synchronize() == 0
    for _ in range(5):
        for w, st, (o, l, ws, need) in zip(worlds, streams, outs):
            mdx.paged_attention(w.cache, w.batch, w.d["q"], o, ws, need, lse=l, stream=st)
    for (o, l, _, _), (a, b) in zip(outs, alone):
        assert np.array_equal(o.get(), a) and np.array_equal(l.get(), b)
    for st in streams:
        assert H.hipStreamDestroy(st) == 0


def test_attention_without_lse_gives_the_same(mdx, gpu):
    rng = np.random.default_rng(14)
    for new, kv in (([1, 1], [600, 40]), ([40, 3], [60, 33])):
        w = World(rng, "fp16", 4, 2, 128, 32, new, kv).upload(mdx)
        a, _ = w.attention(mdx)
        b, _ = w.attention(mdx, want_lse=False)
        assert np.array_equal(a, b)


def test_attention_does_not_depend_on_the_batch_around(mdx, gpu):
    """Again on the same inputs: the same bits."""
    rng = np.random.default_rng(15)
    w = World(rng, "bf16", 4, 1, 128, 16, [1, 40, 1, 200], [3000, 41, 77, 1000]).upload(mdx)
    a, b = w.attention(mdx), w.attention(mdx)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


# ---- append ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("norms", [True, False])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
def test_append(mdx, gpu, nq, nkv, hd, norms, style, dtype):
    rng = np.random.default_rng(nq + hd + style)
    new, kv, max_pos = [1, 5, 0, 37, 3], [1, 20, 9, 64, 2], 5000
    w = World(rng, dtype, nq, nkv, hd, 16, new, kv)
    w.mass += 1
    w.upload(mdx)
    width = (nq + 2 * nkv) * hd
    qkv = rng.standard_normal((w.T, width)).astype(np.float32) * 3
    positions = rng.integers(0, max_pos, w.T).astype(np.int32)
    positions[0], positions[1] = 0, max_pos - 1
    ang = np.arange(max_pos)[:, None] * 1e6 ** (-np.arange(0, hd, 2) / hd)
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    qn, kn = ((1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32) if norms else (None, None))
    dev = [Dev(mdx, x) for x in (qkv, positions, cos, sin)]
    dn = [None if x is None else Dev(mdx, x) for x in (qn, kn)]
    qo = Dev(mdx, np.full((w.T, nq, hd), 0x1111, np.uint16))
    mdx.paged_append(w.cache, w.batch, *dev, max_pos, qo, q_norm=dn[0], k_norm=dn[1], eps=1e-6, rope_style=style)
    q, dq, k, dk, v = ref_append(w, qkv, positions, qn, kn, 1e-6, cos, sin, style)
    assert near(qo.get(), q, dq, dtype) <= 0
    gk, gv, gm, gp = (w.d[n].get() for n in ("k", "v", "mass", "pos"))
    touched = np.zeros((w.n_pages, w.page), bool)
    for r in range(w.R):
        for t, _, row in w.rows(r):
            if row < 0:
                continue
            pg, slot = w.table[r, row // 16], row % 16
            touched[pg, slot] = True
            assert near(gk[pg, :, slot], k[t], dk[t], dtype) <= 0
            assert np.array_equal(gv[pg, :, slot], to16(v[t].astype(np.float32), dtype))
            assert np.all(gm[pg, :, slot] == 0) and np.all(gp[pg, :, slot] == positions[t])
    for got, had in ((gk, w.k), (gv, w.v), (gm, w.mass), (gp, w.pos)):
        assert np.array_equal(got.swapaxes(1, 2)[~touched], had.swapaxes(1, 2)[~touched])


def test_append_leaves_out(mdx, gpu):
    """Positions outside the tables, rows behind the last request, past max_q_len or max_kv_len, pages that do not
    exist, strided rows, a cache without mass and pos."""
    rng = np.random.default_rng(3)
    new, kv, hd, nq, nkv = [4, 6], [40, 30], 64, 2, 1
    w = World(rng, "fp16", nq, nkv, hd, 16, new, kv, max_q=5, max_kv=39)
    w.table[1, 1] = w.n_pages
    w.upload(mdx)
    c = mdx.paged_cache("fp16", nq, nkv, hd, 16, w.n_pages, w.d["k"], w.d["v"])
    T, width = w.T + 2, (nq + 2 * nkv) * hd
    qkv = rng.standard_normal((T, width + 4)).astype(np.float32)
    positions = np.array([3, -1, 9, 10, 4, 5, 10, 2 ** 31 - 1, 8, 1, 2, 2], np.int32)
    ang = np.arange(10)[:, None] * 1e4 ** (-np.arange(0, hd, 2) / hd)
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    b = mdx.paged_batch(w.R, T, w.max_q, w.max_kv, w.max_pages, w.d["q_start"], w.d["kv_len"], w.d["table"])
    dev = [Dev(mdx, x) for x in (qkv, positions, cos, sin)]
    qo = Dev(mdx, np.full((T, nq * hd + 8), 0x1111, np.uint16))
    mdx.paged_append(c, b, *dev, 10, qo, rope_style=1, qkv_stride=width + 4, q_stride=nq * hd + 8)
    w.T, w.q_start[-1] = T, T
    q, dq, k, dk, v = ref_append(w, np.ascontiguousarray(qkv[:, :width]), np.clip(positions, 0, 9), None, None, 1e-6, cos, sin, 1)
    o, gk = qo.get(), w.d["k"].get()
    done = np.array([0, 2, 4, 5, 8])                      # in the tables, within 5 rows of its request
    assert near(o[done, :nq * hd].reshape(-1, nq, hd), q[done], dq[done], "fp16") <= 0
    rest = np.setdiff1d(np.arange(T), done)
    assert np.all(o[rest] == 0x1111) and np.all(o[:, nq * hd:] == 0x1111)
    expect = w.k.copy()
    for t, r, row in ((0, 0, 36), (2, 0, 38)):            # request 1's rows lie in the page that is not there
        pg, slot = w.table[r, row // 16], row % 16
        assert near(gk[pg, :, slot], k[t], dk[t], "fp16") <= 0
        expect[pg, :, slot] = gk[pg, :, slot]
    assert np.array_equal(gk, expect)
    assert np.array_equal(w.d["mass"].get(), w.mass) and np.array_equal(w.d["pos"].get(), w.pos)


# ---- mass ----------------------------------------------------------------------------------

def _check_mass(mdx, w, lse, scale=0.0):
    w.upload(mdx)
    dl = Dev(mdx, lse)
    need = mdx.paged_mass_workspace(w.cache, w.batch)
    ws = Dev(mdx, np.full(max(need, 16), 0xff, np.uint8))
    mdx.paged_mass(w.cache, w.batch, w.d["q"], dl, ws, need, scale=scale)
    got = w.d["mass"].get()
    ref, slack = w.ref_mass(lse.astype(np.float64), scale or None)
    fin = np.isfinite(ref)
    assert np.array_equal(np.isnan(ref), np.isnan(got))
    assert np.array_equal(got[~fin], ref[~fin].astype(np.float32), equal_nan=True)
    assert np.all((np.abs(got - ref) - slack)[fin] <= 0)
    untouched = np.ones(w.mass.shape, bool)
    for r in range(w.R):
        _, pg, slot, ok = w.where(r)
        untouched[pg[ok], :, slot[ok]] = False
    assert np.array_equal(got[untouched], w.mass[untouched])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("new,kv", [([1] * 8, [1, 15, 16, 17, 63, 64, 65, 300]), ([37, 1, 3, 130, 0], [90, 333, 2, 200, 50])])
def test_mass(mdx, gpu, nq, nkv, hd, new, kv, dtype):
    rng = np.random.default_rng(nq + hd)
    w = World(rng, dtype, nq, nkv, hd, 16, new, kv)
    _check_mass(mdx, w, w.ref_attention()[1].astype(np.float32))


@pytest.mark.parametrize("page", [16, 64, 256])
def test_mass_long_chunk(mdx, gpu, page):
    rng = np.random.default_rng(page)
    w = World(rng, "fp16", 4, 2, 64, page, [300, 1], [900, 2000])
    _check_mass(mdx, w, w.ref_attention()[1].astype(np.float32))
    w = World(rng, "bf16", 4, 1, 128, page, [300, 1], [900, 2000], max_q=200, max_kv=850)
    _check_mass(mdx, w, np.full((w.T, 4), 5.0, np.float32), scale=0.05)


def test_mass_of_rows_without_weight(mdx, gpu):
    """lse of -inf (a row that saw nothing) adds nothing; NaN stays with the keys its row sees; pages that do not exist
    and NaN keys that nobody sees are left alone."""
    rng = np.random.default_rng(4)
    w = World(rng, "fp16", 2, 1, 64, 16, [20, 1, 1], [50, 40, 33])
    lse = w.ref_attention()[1].astype(np.float32)
    lse[3], lse[7, 0], lse[20, 1] = -np.inf, np.nan, -np.inf
    w.table[1, 1] = -1
    pg = w.table[0, 3]
    w.k[pg, :, 2:] = to16(np.float32(np.nan), "fp16")         # rows 50.. of request 0's last page
    _check_mass(mdx, w, lse)


# ---- evict -----------------------------------------------------------------------------------

def _evict(mdx, w, budget, sink, recent, in_place):
    w.upload(mdx)
    mo0, po0 = (w.mass, w.pos) if in_place else (np.full(w.mass.shape, -3.0, np.float32), np.full(w.pos.shape, -9, np.int32))
    mo, po = (w.d["mass"], w.d["pos"]) if in_place else (Dev(mdx, mo0), Dev(mdx, po0))
    need = mdx.paged_evict_workspace(w.cache, w.batch, budget)
    ws = Dev(mdx, np.full(need + 64, 0xee, np.uint8))
    mdx.paged_evict(w.cache, w.batch, budget, sink, recent, mo, po, ws, need)
    got = w.d["k"].get(), w.d["v"].get(), mo.get(), po.get()
    assert np.all(ws.get()[need:] == 0xee)
    for a, b in zip(got, w.ref_evict(budget, sink, recent, mo0, po0)):
        assert np.array_equal(a.view(np.uint32) if a.dtype == np.float32 else a, b.view(np.uint32) if b.dtype == np.float32 else b)
    if not in_place:
        assert np.array_equal(w.d["mass"].get().view(np.uint32), w.mass.view(np.uint32)) and np.array_equal(w.d["pos"].get(), w.pos)


def _positions(w, rng, shuffled):
    for r in range(w.R):
        _, pg, slot, _ = w.where(r)
        for h in range(w.nkv):
            w.pos[pg, h, slot] = rng.permutation(len(pg)) if shuffled else np.arange(len(pg))


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("budget,sink,recent", [(64, 4, 16), (1, 0, 0), (1, 1, 0), (0, 0, 0), (100, 0, 0), (100, 50, 50), (257, 1, 256), (1500, 4, 200)])
@pytest.mark.parametrize("dtype,nkv,hd,page", [("fp16", 2, 64, 16), ("bf16", 1, 128, 64), ("fp16", 3, 256, 32)])
def test_evict(mdx, gpu, dtype, nkv, hd, page, budget, sink, recent, in_place):
    rng = np.random.default_rng(budget + hd)
    kv = [1, 63, 64, 65, 100, 101, 257, 1024, 1025, 1600, 0, 2600]
    w = World(rng, dtype, nkv, nkv, hd, page, [0] * len(kv), kv)
    w.mass = np.exp(2 * rng.standard_normal(w.mass.shape)).astype(np.float32)
    _positions(w, rng, shuffled=in_place)
    _evict(mdx, w, budget, sink, recent, in_place)


@pytest.mark.parametrize("what", ["equal", "few values", "zeros", "nan", "inf", "negative"])
def test_evict_ties_and_odd_masses(mdx, gpu, what):
    """Ties go to the lower row, a NaN is the least, zeros of either sign are alike."""
    rng = np.random.default_rng(len(what))
    w = World(rng, "fp16", 2, 2, 64, 16, [0] * 3, [300, 2100, 65])
    m = rng.random(w.mass.shape).astype(np.float32)
    if what == "equal":
        m[:] = 0.25
    elif what == "few values":
        m = np.round(m * 4).astype(np.float32)
    elif what == "zeros":
        m = np.where(m < 0.5, np.float32(0.0), np.float32(-0.0))
    elif what == "nan":
        m[m < 0.9] = np.nan
        m[(m > 0.95)] = -1.0
    elif what == "inf":
        m[m < 0.3], m[m > 0.7] = -np.inf, np.inf
    else:
        m -= 0.5
    w.mass = m
    _positions(w, rng, True)
    _evict(mdx, w, 64, 3, 20, True)


@pytest.mark.parametrize("kv,budget,recent", [([4096, 4097, 4100], 4000, 100), ([16384, 16383, 70], 64, 10), ([16385, 300], 5000, 700), ([40001, 2], 9, 0)])
def test_evict_lengths_of_each_variant(mdx, gpu, kv, budget, recent):
    """Rows per thread: 4, 16 and any number."""
    rng = np.random.default_rng(kv[0])
    w = World(rng, "fp16", 1, 1, 64, 64, [0] * len(kv), kv)
    w.mass = np.round(8 * rng.random(w.mass.shape) ** 4, 2).astype(np.float32)
    _positions(w, rng, True)
    _evict(mdx, w, budget, 4, recent, True)


def test_evict_takes_the_most_recent_by_position(mdx, gpu):
    """Positions far from the rows' numbers, at the ends of their type."""
    rng = np.random.default_rng(1)
    w = World(rng, "bf16", 1, 1, 64, 16, [0], [200])
    _, pg, slot, _ = w.where(0)
    w.pos[pg, 0, slot] = rng.permutation(np.concatenate([np.arange(100), 2 ** 31 - 1 - np.arange(100)]))
    _evict(mdx, w, 60, 10, 30, True)
    w.pos[pg, 0, slot] = 7                                     # all alike: all recent, ties to the lower row
    _evict(mdx, w, 60, 0, 1, True)


# ---- together ----------------------------------------------------------------------------------

def test_steps_together(mdx, gpu):
    """Two requests through a prompt's chunks, single tokens and an eviction, each step against float64 on the cache as
    the device has it."""
    rng = np.random.default_rng(21)
    nq, nkv, hd, page, budget = 4, 2, 64, 16, 48
    w = World(rng, "fp16", nq, nkv, hd, page, [0, 0], [0, 0], extra_pages=12)
    order = rng.permutation(w.n_pages)
    w.max_pages, w.table = 6, order[:12].reshape(2, 6).astype(np.int32)
    w.max_kv, w.R = 6 * page, 2
    ang = np.arange(200)[:, None] * 1e4 ** (-np.arange(0, hd, 2) / hd)
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    qn, kn = (1 + 0.2 * rng.standard_normal((2, hd))).astype(np.float32)
    dcos, dsin, dqn, dkn = (Dev(mdx, x) for x in (cos, sin, qn, kn))
    seen, held = [0, 0], [0, 0]                               # positions so far, rows in the cache
    for step, new in enumerate([[30, 1], [20, 33], [1, 1], [1, 40], [1, 1], [1, 0]]):
        w.new, w.T, w.max_q = new, sum(new), max(new)
        w.q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        held = [h + n for h, n in zip(held, new)]
        w.kv, w.kv_len = list(held), np.asarray(held, np.int32)
        w.q = np.zeros((w.T, nq, hd), np.uint16)
        w.upload(mdx)
        qkv = rng.standard_normal((w.T, (nq + 2 * nkv) * hd)).astype(np.float32) * 2
        positions = np.concatenate([s + np.arange(n) for s, n in zip(seen, new)]).astype(np.int32)
        dx, dp = Dev(mdx, qkv), Dev(mdx, positions)
        mdx.paged_append(w.cache, w.batch, dx, dp, dcos, dsin, 200, w.d["q"], q_norm=dqn, k_norm=dkn, rope_style=1)
        q, dq, k, dk, v = ref_append(w, qkv, positions, qn, kn, 1e-6, cos, sin, 1)
        w.q, w.k, w.v, w.mass, w.pos = (w.d[n].get() for n in ("q", "k", "v", "mass", "pos"))
        assert near(w.q, q, dq, "fp16") <= 0
        for r in range(2):
            for t, _, row in w.rows(r):
                pg, slot = w.table[r, row // page], row % page
                assert near(w.k[pg, :, slot], k[t], dk[t], "fp16") <= 0 and np.all(w.pos[pg, :, slot] == positions[t])
        _, lse = _check_attention(mdx, w)
        ref, slack = w.ref_mass(lse.astype(np.float64))
        dl = Dev(mdx, lse)
        ws = Dev(mdx, np.zeros(max(mdx.paged_mass_workspace(w.cache, w.batch), 16), np.uint8))
        mdx.paged_mass(w.cache, w.batch, w.d["q"], dl, ws, ws.a.nbytes)
        w.mass = w.d["mass"].get()
        assert np.all(np.abs(w.mass - ref) <= slack)
        seen = [s + n for s, n in zip(seen, new)]
        if step >= 2:
            k, v, mo, po = w.ref_evict(budget, 2, 16, w.mass, w.pos)
            ws = Dev(mdx, np.zeros(mdx.paged_evict_workspace(w.cache, w.batch, budget), np.uint8))
            mdx.paged_evict(w.cache, w.batch, budget, 2, 16, w.d["mass"], w.d["pos"], ws, ws.a.nbytes)
            w.k, w.v, w.mass, w.pos = (w.d[n].get() for n in ("k", "v", "mass", "pos"))
            assert all(np.array_equal(a, b) for a, b in ((w.k, k), (w.v, v), (w.mass, mo), (w.pos, po)))
            held = [min(h, budget) for h in held]
    assert held == [budget, budget] and seen == [54, 76]


def test_pool_beyond_32_bits(mdx, gpu):
    """Pages whose values lie more than 2^31 values and 2^32 bytes into the pool, through all four calls."""
    rng = np.random.default_rng(23)
    nq, nkv, hd, page, budget = 8, 8, 128, 1024, 40
    w = World(rng, "bf16", nq, nkv, hd, page, [1, 70], [600, 90], extra_pages=0)
    w.mass = rng.random(w.mass.shape).astype(np.float32)
    w.upload(mdx)
    off = 2100                                             # 2100 pages of 2 MiB
    n = off + w.n_pages
    L = mdx.lib()
    big = {}
    try:
        for name in ("k", "v", "mass", "pos"):
            big[name] = C.c_void_p()
            per = w.d[name].a.nbytes // w.n_pages
            assert L.mdx_device_malloc(C.byref(big[name]), n * per) == 0
            assert L.mdx_memcpy_h2d(big[name].value + off * per, w.d[name].a.ctypes.data, w.d[name].a.nbytes) == 0
        cache = mdx.paged_cache("bf16", nq, nkv, hd, page, n, *(big[x].value for x in ("k", "v", "mass", "pos")))
        table = Dev(mdx, np.where(w.table >= 0, w.table + off, -1).astype(np.int32))
        batch = mdx.paged_batch(w.R, w.T, w.max_q, w.max_kv, w.max_pages, w.d["q_start"], w.d["kv_len"], table)

        def pages(name):
            a = np.empty_like(w.d[name].a)
            assert L.mdx_device_synchronize() == 0
            assert L.mdx_memcpy_d2h(a.ctypes.data, big[name].value + off * (a.nbytes // w.n_pages), a.nbytes) == 0
            return a

        out, lse = Dev(mdx, np.zeros(w.q.shape, np.uint16)), Dev(mdx, np.zeros((w.T, nq), np.float32))
        need = max(mdx.paged_attention_workspace(cache, batch), mdx.paged_mass_workspace(cache, batch), mdx.paged_evict_workspace(cache, batch, budget))
        ws = Dev(mdx, np.zeros(max(need, 16), np.uint8))
        qkv = rng.standard_normal((w.T, (nq + 2 * nkv) * hd)).astype(np.float32)
        positions = np.concatenate([[599], np.arange(20, 90)]).astype(np.int32)
        cos, sin = np.ones((600, hd // 2), np.float32), np.zeros((600, hd // 2), np.float32)
        dev = [Dev(mdx, x) for x in (qkv, positions, cos, sin)]
        mdx.paged_append(cache, batch, *dev, 600, w.d["q"])
        w.q, w.k, w.v, w.mass, w.pos = w.d["q"].get(), pages("k"), pages("v"), pages("mass"), pages("pos")
        _, _, k, dk, v = ref_append(w, qkv, positions, None, None, 0.0, cos, sin, 0)
        for r in range(2):
            for t, _, row in w.rows(r):
                pg, slot = w.table[r, row // page], row % page
                assert near(w.k[pg, :, slot], k[t], dk[t], "bf16") <= 0 and np.array_equal(w.v[pg, :, slot], to16(v[t].astype(np.float32), "bf16"))
        mdx.paged_attention(cache, batch, w.d["q"], out, ws, ws.a.nbytes, lse=lse)
        ref, _, slack, _ = w.ref_attention()
        assert near(out.get(), ref, slack, "bf16") <= 0
        mdx.paged_mass(cache, batch, w.d["q"], lse, ws, ws.a.nbytes)
        mass, slack = w.ref_mass(lse.get().astype(np.float64))
        w.mass = pages("mass")
        assert np.all(np.abs(w.mass - mass) <= slack)
        mdx.paged_evict(cache, batch, budget, 2, 10, big["mass"].value, big["pos"].value, ws, ws.a.nbytes)
        want = w.ref_evict(budget, 2, 10, w.mass, w.pos)
        assert all(np.array_equal(pages(x), y) for x, y in zip(("k", "v", "mass", "pos"), want))
    finally:
        for x in big.values():
            L.mdx_device_free(x)


def _hip():
    from test_zz_no_alloc import _hip as f
    return f()


def test_captured_chunks(mdx, gpu):
    """A chunk's attention and mass from one captured graph, replayed with other lengths of chunk and cache."""
    L, H = mdx.lib(), _hip()
    rng = np.random.default_rng(24)
    w = World(rng, "fp16", 4, 2, 128, 32, [200, 40], [900, 700]).upload(mdx)
    out, lse = Dev(mdx, np.zeros(w.q.shape, np.uint16)), Dev(mdx, np.zeros((w.T, 4), np.float32))
    sizes = mdx.paged_attention_workspace(w.cache, w.batch), mdx.paged_mass_workspace(w.cache, w.batch)
    ws = [Dev(mdx, np.full(max(n, 16), 0xff, np.uint8)) for n in sizes]
    stream, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert H.hipStreamCreate(C.byref(stream)) == 0
    try:
        w.attention(mdx)                                   # a first call outside the capture
        assert H.hipStreamBeginCapture(stream, 2) == 0
        mdx.paged_attention(w.cache, w.batch, w.d["q"], out, ws[0], sizes[0], lse=lse, stream=stream)
        mdx.paged_mass(w.cache, w.batch, w.d["q"], lse, ws[1], sizes[1], stream=stream)
        assert H.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert H.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
        for new, kv in (([200, 40], [900, 700]), ([1, 200], [900, 333]), ([17, 3], [17, 700]), ([0, 130], [5, 130])):
            w.new, w.kv = new, kv
            w.q_start, w.kv_len = np.array([0, new[0], sum(new)], np.int32), np.array(kv, np.int32)
            w.d["q_start"].put(w.q_start)
            w.d["kv_len"].put(w.kv_len)
            w.d["mass"].put(w.mass)
            assert L.mdx_device_synchronize() == 0
            assert H.hipGraphLaunch(exe, stream) == 0
            assert H.hipStreamSynchronize(stream) == 0
            ref, rlse, slack, lslack = w.ref_attention()
            n = sum(new)
            got = lse.get()
            assert near(out.get()[:n], ref[:n], slack[:n], "fp16") <= 0 and np.all(np.abs(got - rlse)[:n] <= lslack[:n])
            mass, ms = w.ref_mass(got.astype(np.float64))
            assert np.all(np.abs(w.d["mass"].get() - mass) <= ms)
            w.attention(mdx)                               # other work between the replays
    finally:
        if exe.value:
            H.hipGraphExecDestroy(exe)
        if graph.value:
            H.hipGraphDestroy(graph)
        H.hipStreamDestroy(stream)


def test_captured_steps(mdx, gpu):
    """A step of all four calls on a stream, captured, replayed with other rows, lengths and tables in the same arrays;
    every replay against the eager calls on a copy of the pool."""
    L, H = mdx.lib(), _hip()
    rng = np.random.default_rng(22)
    nq, nkv, hd, page, R, budget = 4, 2, 64, 16, 3, 600
    w = World(rng, "bf16", nq, nkv, hd, page, [1] * R, [700] * R).upload(mdx)
    e = World(np.random.default_rng(22), "bf16", nq, nkv, hd, page, [1] * R, [700] * R).upload(mdx)
    ang = np.arange(1000)[:, None] * 1e4 ** (-np.arange(0, hd, 2) / hd)
    tabs = [Dev(mdx, f(ang).astype(np.float32)) for f in (np.cos, np.sin)]
    qkv, positions = Dev(mdx, np.zeros((R, (nq + 2 * nkv) * hd), np.float32)), Dev(mdx, np.zeros(R, np.int32))
    bufs = {}
    for x in (w, e):
        sizes = mdx.paged_attention_workspace(x.cache, x.batch), mdx.paged_mass_workspace(x.cache, x.batch), mdx.paged_evict_workspace(x.cache, x.batch, budget)
        bufs[x] = (Dev(mdx, np.zeros((R, nq, hd), np.uint16)), Dev(mdx, np.zeros((R, nq), np.float32)), [Dev(mdx, np.zeros(max(n, 16), np.uint8)) for n in sizes])

    def step(x, stream):
        out, lse, ws = bufs[x]
        mdx.paged_append(x.cache, x.batch, qkv, positions, *tabs, 1000, x.d["q"], rope_style=0, stream=stream)
        mdx.paged_attention(x.cache, x.batch, x.d["q"], out, ws[0], ws[0].a.nbytes, lse=lse, stream=stream)
        mdx.paged_mass(x.cache, x.batch, x.d["q"], lse, ws[1], ws[1].a.nbytes, stream=stream)
        mdx.paged_evict(x.cache, x.batch, budget, 4, 100, x.d["mass"], x.d["pos"], ws[2], ws[2].a.nbytes, stream=stream)

    stream, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert H.hipStreamCreate(C.byref(stream)) == 0
    try:
        step(e, None)                                       # a first call outside the capture
        for n in ("k", "v", "mass", "pos"):
            e.d[n].put(getattr(w, n))
        assert H.hipStreamBeginCapture(stream, 2) == 0
        step(w, stream)
        assert H.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert H.hipGraphInstantiate(C.byref(exe), graph, None, None, C.c_size_t(0)) == 0
        for rep in range(4):
            x, kv = rng.standard_normal(qkv.a.shape).astype(np.float32), rng.integers(1, 700, R).astype(np.int32)
            kv[rep % R] = 700 - rep
            table = np.stack([rng.permutation(w.n_pages)[:w.max_pages] for _ in range(1)]).repeat(R, 0).astype(np.int32)
            perm = rng.permutation(w.n_pages)[:R * w.max_pages].reshape(R, -1).astype(np.int32)
            for y in (w, e):
                y.d["kv_len"].put(kv)
                y.d["table"].put(perm if perm.shape == table.shape else table)
            qkv.put(x)
            positions.put(kv)
            assert L.mdx_device_synchronize() == 0
            assert H.hipGraphLaunch(exe, stream) == 0
            assert H.hipStreamSynchronize(stream) == 0
            step(e, None)
            assert L.mdx_device_synchronize() == 0
            for a, b in zip(bufs[w][:2], bufs[e][:2]):
                assert np.array_equal(a.get(), b.get()), rep
            for n in ("k", "v", "mass", "pos", "q"):
                assert np.array_equal(w.d[n].get(), e.d[n].get()), (rep, n)
    finally:
        if exe.value:
            H.hipGraphExecDestroy(exe)
        if graph.value:
            H.hipGraphDestroy(graph)
        H.hipStreamDestroy(stream)
