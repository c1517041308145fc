"""The paged cache's operators in float64 numpy, and arrays on the device for
their entry points.

Conversions to fp16 / bf16 round to nearest even.  A `World` is a pool of pages
with requests in it: random K/V rows everywhere (also behind the last row of a
request), pages in any order, -1 behind a request's pages."""
from __future__ import annotations

import ctypes as C

import numpy as np

EPS = {"fp16": 2.0 ** -10, "bf16": 2.0 ** -7}       # finfo(t).eps
TINY = {"fp16": 2.0 ** -24, "bf16": 2.0 ** -133}    # the smallest number above 0


def to16(x, dtype):
    """fp32 values as the bits of `dtype`."""
    x = np.asarray(x, np.float32)
    if dtype == "fp16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    b = ((u + np.uint32(0x7fff) + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), b)


def wide(bits, dtype):
    """The float64 values of 16-bit numbers."""
    bits = np.asarray(bits, np.uint16)
    if dtype == "fp16":
        return bits.view(np.float16).astype(np.float64)
    return (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class Dev:
    """A numpy array's copy in device memory."""

    def __init__(self, mdx, a):
        self.L, self.a = mdx.lib(), np.ascontiguousarray(a)
        self.p = C.c_void_p()
        assert self.L.mdx_device_malloc(C.byref(self.p), max(self.a.nbytes, 256)) == 0
        self.put(self.a)

    def put(self, a):
        a = np.ascontiguousarray(a, self.a.dtype)
        assert a.nbytes == self.a.nbytes and self.L.mdx_memcpy_h2d(self.p, a.ctypes.data, a.nbytes) == 0

    def get(self):
        out = np.empty_like(self.a)
        assert self.L.mdx_device_synchronize() == 0
        assert self.L.mdx_memcpy_d2h(out.ctypes.data, self.p, out.nbytes) == 0
        return out

    def data_ptr(self):
        return self.p.value

    def __del__(self):
        self.L.mdx_device_free(self.p)


class World:
    def __init__(self, rng, dtype, nq, nkv, hd, page, new, kv, extra_pages=2, std=1.0, max_q=None, max_kv=None, q_std=1.5):
        self.dtype, self.nq, self.nkv, self.hd, self.page = dtype, nq, nkv, hd, page
        self.G, self.new, self.kv = nq // nkv, list(new), list(kv)
        self.R, self.T = len(new), sum(new)
        used = [-(-n // page) for n in kv]
        self.n_pages, self.max_pages = sum(used) + extra_pages, max(used + [1])
        order = rng.permutation(self.n_pages)
        self.table = np.full((self.R, self.max_pages), -1, np.int32)
        at = 0
        for r, n in enumerate(used):
            self.table[r, :n] = order[at:at + n]
            at += n
        self.q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.kv_len = np.asarray(kv, np.int32)
        self.max_q = max(list(new) + [0]) if max_q is None else max_q
        self.max_kv = max(list(kv) + [0]) if max_kv is None else max_kv
        shape = (self.n_pages, nkv, page, hd)
        self.k = to16(rng.standard_normal(shape) * std, dtype)
        self.v = to16(rng.standard_normal(shape) * std, dtype)
        self.q = to16(rng.standard_normal((self.T, nq, hd)) * q_std, dtype)
        self.mass = rng.random((self.n_pages, nkv, page)).astype(np.float32)
        self.pos = np.zeros((self.n_pages, nkv, page), np.int32)

    # ---- device side
    def upload(self, mdx, T=None):
        self.d = {n: Dev(mdx, getattr(self, n)) for n in ("k", "v", "q", "mass", "pos", "table", "q_start", "kv_len")}
        self.cache = mdx.paged_cache(self.dtype, self.nq, self.nkv, self.hd, self.page, self.n_pages, self.d["k"], self.d["v"],
                                     self.d["mass"], self.d["pos"])
        self.batch = mdx.paged_batch(self.R, self.T if T is None else T, self.max_q, self.max_kv, self.max_pages, self.d["q_start"], self.d["kv_len"],
                                     self.d["table"])
        return self

    def attention(self, mdx, scale=0.0, want_lse=True, stream=None):
        """(out, lse) of the device; both start as a pattern that has to go."""
        out = Dev(mdx, np.full(self.q.shape, 0x3555, np.uint16))
        lse = Dev(mdx, np.full((self.T, self.nq), 77.0, np.float32)) if want_lse else None
        need = mdx.paged_attention_workspace(self.cache, self.batch)
        ws = Dev(mdx, np.full(max(need, 16), 0xff, np.uint8))         # NaN everywhere
        mdx.paged_attention(self.cache, self.batch, self.d["q"], out, ws, need, lse=lse, scale=scale, stream=stream)
        return out.get(), (lse.get() if want_lse else None)

    # ---- reference
    def where(self, r):
        """(page, row) of the cache rows of request r that exist."""
        n = max(0, min(self.kv[r], self.max_kv, self.max_pages * self.page))
        j = np.arange(n)
        pg = self.table[r, j // self.page] if n else np.zeros(0, np.int32)
        return j, pg, j % self.page, (pg >= 0) & (pg < self.n_pages)

    def rows(self, r):
        """(batch row, i, cache row) of request r's new rows that take part."""
        for i in range(min(self.new[r], self.max_q)):
            yield self.q_start[r] + i, i, self.kv[r] - self.new[r] + i

    def ref_attention(self, scale=None):
        """out, lse in float64 and, per output, the bound of its error beside its own rounding."""
        scale = 1 / np.sqrt(self.hd) if scale is None else scale
        q = wide(self.q, self.dtype)
        out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
        slack, lse_slack = np.zeros(q.shape), np.zeros(q.shape[:2])
        with np.errstate(all="ignore"):
            for r in range(self.R):
                j, pg, slot, ok = self.where(r)
                j, pg, slot = j[ok], pg[ok], slot[ok]
                k, v = wide(self.k[pg, :, slot], self.dtype), wide(self.v[pg, :, slot], self.dtype)
                for t, _, row in self.rows(r):
                    m = int(np.searchsorted(j, row, side="right"))
                    if m == 0:
                        continue
                    for h in range(self.nq):
                        kk, vv = k[:m, h // self.G], v[:m, h // self.G]
                        s = scale * (kk @ q[t, h])
                        # IEEE: the maximum looks past NaN, everything after it carries them
                        top = np.fmax.reduce(s)
                        p = np.exp(s - top)
                        out[t, h] = (p[:, None] * vv).sum(0) / p.sum()
                        lse[t, h] = top + np.log(p.sum()) if np.isfinite(top) else (top if not np.isnan(s).any() and top < 0 else np.nan)
                        # a score's fp32 sum over hd exact products, and its exponent's roundings
                        reach = scale * np.abs(kk * q[t, h]).sum(1).max()
                        ds = (self.hd * reach + 2 * np.abs(s - top).max() + 16) * 2.0 ** -23
                        share = (p[:, None] * np.abs(vv)).sum(0) / p.sum()
                        # a probability's rounding to the type (half a step, and half the smallest
                        # number beside the largest one), and m fp32 additions
                        slack[t, h] = (EPS[self.dtype] / 2 + 2 * ds + m * 2.0 ** -23) * share + TINY[self.dtype] / 2 * np.abs(vv).sum(0)
                        lse_slack[t, h] = 2 * ds + m * 2.0 ** -24 + 2.0 ** -22 * (abs(top) + abs(lse[t, h]) + 8)
        return out, lse, slack, lse_slack

    def ref_mass(self, lse, scale=None):
        """mass in float64 after the call, and the bound of its error."""
        scale = 1 / np.sqrt(self.hd) if scale is None else scale
        q, mass = wide(self.q, self.dtype), self.mass.astype(np.float64)
        slack = np.abs(mass) * 2.0 ** -24
        for r in range(self.R):
            j, pg, slot, ok = self.where(r)
            j, pg, slot = j[ok], pg[ok], slot[ok]
            k = wide(self.k[pg, :, slot], self.dtype)
            add, rough = np.zeros((len(j), self.nkv)), np.zeros((len(j), self.nkv))
            for t, _, row in self.rows(r):
                m = int(np.searchsorted(j, row, side="right"))
                for h in range(self.nq):
                    if m == 0 or lse[t, h] == -np.inf:
                        continue
                    s = scale * (k[:m, h // self.G] @ q[t, h])
                    w = np.exp(s - lse[t, h])
                    reach = scale * np.abs(k[:m, h // self.G] * q[t, h]).sum(1)
                    add[:m, h // self.G] += w
                    rough[:m, h // self.G] += w * (self.hd * reach + 2 * np.abs(s - lse[t, h]) + 2 * np.abs(s) + 16) * 2.0 ** -23
            n = sum(self.new) * self.G
            mass[pg, :, slot] += add
            slack[pg, :, slot] += rough + (n * add + np.abs(mass[pg, :, slot])) * 2.0 ** -23
        return mass, slack

    def ref_evict(self, budget, sink, recent, mass_out, pos_out):
        """k, v, mass_out, pos_out after the call."""
        k, v, mo, po = self.k.copy(), self.v.copy(), mass_out.copy(), pos_out.copy()
        for r in range(self.R):
            j, pg, slot, ok = self.where(r)
            assert ok.all()
            n = len(j)
            for h in range(self.nkv):
                m, p = self.mass[pg, h, slot], self.pos[pg, h, slot]
                first = slice(0, min(n, budget))
                if n <= budget:
                    mo[pg[first], h, slot[first]], po[pg[first], h, slot[first]] = m, p
                    continue
                safe = (p < sink) | (p.astype(np.int64) > int(p.max()) - recent)
                order = sorted(range(n), key=lambda x: (not safe[x], 0.0 if safe[x] else (np.inf if np.isnan(m[x]) else -float(m[x])),
                                                        0 if safe[x] or not np.isnan(m[x]) else 1, x))
                stays = np.zeros(n, bool)
                stays[order[:budget]] = True
                gaps, fill = np.flatnonzero(~stays[:budget]), budget + np.flatnonzero(stays[budget:])
                assert len(gaps) == len(fill)
                keep = np.flatnonzero(stays[:budget])
                mo[pg[keep], h, slot[keep]], po[pg[keep], h, slot[keep]] = m[keep], p[keep]
                for to, src in zip(gaps, fill):
                    k[pg[to], h, slot[to]], v[pg[to], h, slot[to]] = self.k[pg[src], h, slot[src]], self.v[pg[src], h, slot[src]]
                    mo[pg[to], h, slot[to]], po[pg[to], h, slot[to]] = m[src], p[src]
        return k, v, mo, po


def ref_append(w, qkv, positions, q_norm, k_norm, eps, cos, sin, style):
    """(q, k of every row, v of every row, bound of q's and k's error beside their rounding), float64 [T][heads][hd]."""
    x = qkv.astype(np.float64).reshape(w.T, w.nq + 2 * w.nkv, w.hd)
    c, s = cos[positions].astype(np.float64)[:, None], sin[positions].astype(np.float64)[:, None]

    def turn(x, norm):
        if norm is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
        a, b = (x[..., 0::2], x[..., 1::2]) if style == 0 else (x[..., :w.hd // 2], x[..., w.hd // 2:])
        y, z, size = a * c - b * s, b * c + a * s, np.abs(a) + np.abs(b)
        if style == 0:
            pair = lambda u, v: np.stack([u, v], -1).reshape(x.shape)  # noqa: E731
        else:
            pair = lambda u, v: np.concatenate([u, v], -1)  # noqa: E731
        # fp32: hd additions under the root (half of their error), the root, four products and a sum
        return pair(y, z), pair(size, size) * (w.hd / 2 + 10) * 2.0 ** -24

    q, dq = turn(x[:, :w.nq], q_norm)
    k, dk = turn(x[:, w.nq:w.nq + w.nkv], k_norm)
    return q, dq, k, dk, x[:, w.nq + w.nkv:]


def near(got_bits, ref, slack, dtype):
    """Largest excess of |got - ref| over half a step of the type plus slack; the same places have to be non-finite."""
    got = wide(got_bits, dtype)
    fin = np.isfinite(ref)
    if not np.array_equal(fin, np.isfinite(got)) or not np.array_equal(np.isnan(ref), np.isnan(got)):
        return np.inf
    if not np.array_equal(got[~fin & ~np.isnan(ref)], ref[~fin & ~np.isnan(ref)]):
        return np.inf
    bound = EPS[dtype] / 2 * (np.abs(ref) + slack) + slack + TINY[dtype] / 2
    return float(np.max(np.abs(got[fin] - ref[fin]) - bound[fin], initial=-1.0))
