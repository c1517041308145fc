"""The paged cache's operators as measurable cases: many requests that share one pool of K/V pages.

Four kinds of passes, each one call of a program that serves requests:

  append     the qkv rows of a step's new tokens: RMSNorm of each query and key head, rotation, K and V into their
             requests' pages, the queries as rows for the attention.
  attention  the new tokens' attention over their requests' pages: one token a request (decoding), chunks of a
             prompt, and both in one batch.
  mass       the attention weight that each cached row has received, added up for each KV head.
  evict      a cache that is over its budget: the rows of least weight go, the ones that stay close the gaps.

The cache is k_pages, v_pages [pages][KV heads][rows of a page][head_dim] and mass, pos [pages][KV heads][rows of a
page].  Row i of a request's n new rows is row kv_len - n + i of its cache and sees the rows up to itself.

The head shapes are the repository's own (16 query heads over 8 KV heads of 128; 8 over 4 of 64; 16 over 4 of 128) and
generic ones.
"""
from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

EPS, THETA = 1e-6, 1e6
SINK = 4                      # rows at the start of a request that are never evicted
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases -----------------------------------------------------------------

def _case(kind, dtype, nq, nkv, hd, page, requests, new, kv, **more):
    """new: the most new rows of a request, and how they are spread ("one", "chunk", "mixed"); kv: the longest cache."""
    spread = more.pop("spread", "one" if new == 1 else "chunk")
    return dict(kind=kind, dtype=dtype, nq=nq, nkv=nkv, hd=hd, page=page, requests=requests, new=new, spread=spread, kv=kv, **more)


def listed():
    return [
        # the smallest call: the next token of one request, where the launch is most of the time
        dict(name="append_1", **_case("append", "fp16", 16, 8, 128, 64, 1, 1, 512, style=1, norm=True)),
        # a step of many requests, some in their prompt, small heads, pairs rotated, no norms
        dict(name="append_mixed_37", **_case("append", "bf16", 8, 4, 64, 16, 37, 61, 700, spread="mixed", style=0, norm=False)),
        # a long prompt's chunk
        dict(name="append_4096", **_case("append", "fp16", 16, 8, 128, 64, 1, 4096, 4096, style=1, norm=True)),
        # the next token of one request with an ordinary context
        dict(name="attn_1x512", **_case("attention", "fp16", 16, 8, 128, 64, 1, 1, 512)),
        # a decoding step of many requests of different lengths
        dict(name="attn_64x4096", **_case("attention", "fp16", 16, 8, 128, 64, 64, 1, 4096)),
        # one request with a very long context
        dict(name="attn_1x131072", **_case("attention", "bf16", 16, 8, 128, 256, 1, 1, 131072)),
        # prompts' chunks next to requests that decode, groups of four query heads
        dict(name="attn_mixed_24", **_case("attention", "bf16", 16, 4, 128, 16, 24, 203, 2000, spread="mixed")),
        # a long prompt's later chunk: the matrix products are what takes the time
        dict(name="attn_2048_over_8192", **_case("attention", "fp16", 16, 8, 128, 64, 1, 2048, 8192)),
        # weights of a decoding step, contexts a little over a budget
        dict(name="mass_32x2049", **_case("mass", "fp16", 16, 8, 128, 64, 32, 1, 2049)),
        # weights of a prompt's last chunk, small heads
        dict(name="mass_515_over_4000", **_case("mass", "bf16", 8, 4, 64, 32, 2, 515, 4000)),
        # the steady state: every request one row over its budget
        dict(name="evict_32x2049", **_case("evict", "fp16", 16, 8, 128, 64, 32, 1, 2049, budget=2048, recent=256, even=True)),
        # after long prompts: most rows go
        dict(name="evict_4x16384", **_case("evict", "fp16", 16, 8, 128, 64, 4, 1, 16384, budget=2048, recent=512)),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype, page = rng.choice(["fp16", "bf16"]), rng.choice([16, 32, 64, 128, 256])
    nkv, group, hd = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8]), rng.choice([64, 128, 128, 256])
    heads = (dtype, nkv * group, nkv, hd, page)
    kind = rng.choice(["append", "attention", "attention", "mass", "evict"])
    if kind == "append":
        requests = _spread(rng, 1, 64)
        new = _spread(rng, 1, 4096 // requests)
        return _case("append", *heads, requests, new, new + _spread(rng, 1, 1000), spread=rng.choice(["chunk", "mixed"]),
                     style=rng.randint(0, 1), norm=rng.random() < 0.7)
    if kind == "evict":
        requests, budget = _spread(rng, 1, 16), _spread(rng, 40, 2048)
        return _case("evict", *heads, requests, 1, min(16384, budget + _spread(rng, 1, 8192)), budget=budget, recent=_spread(rng, 1, budget // 2))
    if rng.random() < 0.5:
        requests = _spread(rng, 1, 64)
        return _case(kind, *heads, requests, 1, _spread(rng, 16, 65536 // requests))
    requests, new = _spread(rng, 1, 8), _spread(rng, 2, 1024)
    return _case(kind, *heads, requests, new, new + _spread(rng, 1, 4096), spread=rng.choice(["chunk", "mixed"]))


def _lengths(case):
    """(new rows, rows with them) of each request: the case's own, whatever the seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    R, new, kv = case["requests"], case["new"], case["kv"]
    n = [1 if case["spread"] == "one" or (case["spread"] == "mixed" and rng.random() < 0.6) else rng.randint(1, new) for _ in range(R)]
    n[0] = new
    if case.get("even"):
        return n, [kv] * R
    return n, [kv] + [rng.randint(max(n[r], kv // 4), max(n[r], kv)) for r in range(1, R)]


# ---- inputs ----------------------------------------------------------------------

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    nq, nkv, hd, page, R = (case[k] for k in ("nq", "nkv", "hd", "page", "requests"))
    new, kv = _lengths(case)
    T, most = sum(new), -(-max(kv) // page)
    used = [-(-n // page) for n in kv]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device="cuda")[: sum(used)].tolist()
    table, at = [], 0
    for n in used:
        table.append(order[at:at + n] + [-1] * (most - n))
        at += n
    s = dict(case=case, new=new, kv=kv, T=T, pages=pages, max_pages=most,
             q_start=_ints([0] + list(np.cumsum(new))), kv_len=_ints(kv), table=_ints(table),
             k_pages=randn(pages, nkv, page, hd, dtype=dt), v_pages=randn(pages, nkv, page, hd, dtype=dt))
    if case["kind"] in ("append", "evict", "mass"):
        # weights that rows have gathered so far: a few draw most of it
        s["mass"] = 0.01 * torch.exp(2 * randn(pages, nkv, page))
        s["pos"] = torch.zeros(pages, nkv, page, dtype=torch.int32, device="cuda")
    if case["kind"] == "append":
        positions = [kv[r] - new[r] + i for r in range(R) for i in range(new[r])]
        inv = THETA ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
        angle = torch.arange(max(kv), device="cuda", dtype=torch.float64)[:, None] * inv
        s.update(qkv=randn(T, (nq + 2 * nkv) * hd), positions=_ints(positions), cos=angle.cos().float(), sin=angle.sin().float(),
                 q_norm=1 + 0.1 * randn(hd) if case["norm"] else None, k_norm=1 + 0.1 * randn(hd) if case["norm"] else None,
                 q=torch.zeros(T, nq, hd, dtype=dt, device="cuda"))
    elif case["kind"] in ("attention", "mass"):
        # normed queries and keys: scores of a few units
        s["q"] = randn(T, nq, hd, dtype=dt, std=1.5)
        s["scale"] = 1.0 / math.sqrt(hd)
        if case["kind"] == "mass":
            s["lse"] = _attend(s)[1]
        else:
            s.update(out=torch.zeros(T, nq, hd, dtype=dt, device="cuda"), lse=torch.zeros(T, nq, device="cuda"))
    else:
        # the positions that a cache holds which has been through this before: its rows in any order
        j = torch.argsort(torch.rand(R, nkv, max(kv), generator=g, device="cuda") + 2.0 * (torch.arange(max(kv), device="cuda") >= s["kv_len"][:, None])[:, None], dim=2)
        at, slot = _rows(s)
        s["pos"][at[:, None], torch.arange(nkv, device="cuda")[:, None], slot[:, None]] = torch.where(_held(s)[:, None], j.int(), 0)
        s["mass_out"], s["pos_out"] = torch.zeros_like(s["mass"]), torch.zeros_like(s["pos"])
    return s


# ---- the plain forms -----------------------------------------------------------------

def _rows(s):
    """Page and row in it of every cache row, [R][longest]; rows that a request does not have: the last page of the pool."""
    j = torch.arange(max(s["kv"]), device="cuda")
    page = s["table"][:, j // s["case"]["page"]].long()
    return torch.where(_held(s) & (page >= 0), page, s["pages"] - 1), (j % s["case"]["page"]).expand_as(page)


def _held(s):
    return torch.arange(max(s["kv"]), device="cuda") < s["kv_len"][:, None]


def _new_rows(s):
    """Request, cache row and place in a [R][most new] batch of every new row."""
    t = torch.arange(s["T"], device="cuda")
    r = torch.bucketize(t, s["q_start"][1:], right=True)
    i = t - s["q_start"][r]
    return r, s["kv_len"][r] - (s["q_start"][r + 1] - s["q_start"][r]) + i, i


def _scores(s):
    """Scaled scores [R][nkv][group][most new][longest], -inf where a row does not see, and the index of the new rows."""
    c = s["case"]
    R, G = c["requests"], c["nq"] // c["nkv"]
    r, row, i = _new_rows(s)
    m = max(s["new"])
    q = torch.zeros(R, m, c["nq"], c["hd"], device="cuda")
    q[r, i] = s["q"].float()
    last = torch.full((R, m), -1, device="cuda", dtype=torch.long)
    last[r, i] = row
    at, slot = _rows(s)
    k = s["k_pages"][at, :, slot].float().permute(0, 2, 3, 1)                     # [R][nkv][hd][longest]
    q = q.view(R, m, c["nkv"], G, c["hd"]).permute(0, 2, 3, 1, 4).reshape(R, c["nkv"], G * m, c["hd"])
    w = (torch.matmul(q, k) * s["scale"]).view(R, c["nkv"], G, m, -1)
    seen = torch.arange(max(s["kv"]), device="cuda") <= last[:, :, None]
    return w.masked_fill_(~seen[:, None, None], -math.inf), r, i


def _attend(s):
    c = s["case"]
    w, r, i = _scores(s)
    top = w.amax(-1, keepdim=True).clamp_min(-3e38)
    p = w.sub_(top).exp_()
    l = p.sum(-1, keepdim=True)
    at, slot = _rows(s)
    v = s["v_pages"][at, :, slot].float().masked_fill_(~_held(s)[:, :, None, None], 0.0).permute(0, 2, 1, 3)
    o = torch.matmul(p.flatten(2, 3), v).view(*p.shape[:4], c["hd"]) / l.clamp_min(1e-38)
    lse = (top + l.log()).squeeze(-1)
    rows = lambda x: x.flatten(1, 2).transpose(1, 2)[r, i]  # noqa: E731  [R][nkv][G][m]... -> [T][nq]...
    return rows(o).to(s["q"].dtype), rows(lse)


def _mass(s):
    w, r, i = _scores(s)
    c = s["case"]
    lse = torch.zeros(c["requests"], max(s["new"]), c["nq"], device="cuda")
    lse[r, i] = s["lse"]
    lse = lse.view(*lse.shape[:2], c["nkv"], -1).permute(0, 2, 3, 1)[..., None]
    got = (w - lse).exp_().sum((2, 3))                                             # [R][nkv][longest]
    at, slot = _rows(s)
    before = s["mass"][at, :, slot].transpose(1, 2)
    r, j = _held(s).nonzero(as_tuple=True)
    s["mass"][at[r, j], :, slot[r, j]] = (before + got)[r, :, j]
    return s["mass"]


def _append(s):
    c = s["case"]
    nq, nkv, hd = c["nq"], c["nkv"], c["hd"]
    x = s["qkv"].float().view(s["T"], nq + 2 * nkv, hd)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]

    def turned(x, w):
        if w is not None:
            x = x * (1 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)) * w
        a, b = (x[..., 0::2], x[..., 1::2]) if c["style"] == 0 else (x[..., :hd // 2], x[..., hd // 2:])
        y = [a * cos - b * sin, b * cos + a * sin]
        return torch.stack(y, -1).flatten(-2) if c["style"] == 0 else torch.cat(y, -1)

    dt = s["q"].dtype
    s["q"].copy_(turned(q, s["q_norm"]).to(dt))
    r, row, _ = _new_rows(s)
    page, slot = s["table"][r, row // c["page"]].long(), (row % c["page"]).long()
    s["k_pages"][page, :, slot] = turned(k, s["k_norm"]).to(dt)
    s["v_pages"][page, :, slot] = v.to(dt)
    s["mass"][page, :, slot] = 0.0
    s["pos"][page, :, slot] = s["positions"][:, None].expand(-1, nkv)
    return s["q"], s["k_pages"], s["v_pages"], s["mass"], s["pos"]


def _evict(s):
    c = s["case"]
    at, slot = _rows(s)
    held, budget = _held(s)[:, None], c["budget"]
    mass, pos = s["mass"][at, :, slot].transpose(1, 2), s["pos"][at, :, slot].transpose(1, 2)
    pos = pos.masked_fill(~held, -1)
    newest = pos.amax(-1, keepdim=True)
    kept_anyway = (pos < SINK) | (pos > newest - c["recent"])
    rank = mass.masked_fill(kept_anyway, math.inf).masked_fill(~held, -math.inf)
    best = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    keep = torch.zeros_like(held.expand_as(mass)).scatter_(-1, best, True) & held
    over = (s["kv_len"] > budget)[:, None, None]
    stays = held & (torch.arange(mass.shape[-1], device="cuda") < budget)
    r, h, j = stays.expand_as(keep).nonzero(as_tuple=True)
    s["mass_out"][at[r, j], h, slot[r, j]] = mass[r, h, j]
    s["pos_out"][at[r, j], h, slot[r, j]] = pos[r, h, j]
    r, h, to = (~keep[..., :budget] & over).nonzero(as_tuple=True)
    _, _, src = (keep[..., budget:] & over).nonzero(as_tuple=True)
    src = src + budget
    p, i, p2, i2 = at[r, to], slot[r, to], at[r, src], slot[r, src]
    s["k_pages"][p, h, i], s["v_pages"][p, h, i] = s["k_pages"][p2, h, i2], s["v_pages"][p2, h, i2]
    s["mass_out"][p, h, i], s["pos_out"][p, h, i] = mass[r, h, src], pos[r, h, src]
    return s["k_pages"], s["v_pages"], s["mass_out"], s["pos_out"]


# ---- a pass -------------------------------------------------------------------------

def _handles(s):
    """What a program makes once for its cache, its batch and its workspace."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rknn-matmul-parallel_amd"))
    import mdx_lib as mdx
    c = s["case"]
    cache = mdx.paged_cache(c["dtype"], c["nq"], c["nkv"], c["hd"], c["page"], s["pages"], s["k_pages"], s["v_pages"], s.get("mass"), s.get("pos"))
    batch = mdx.paged_batch(c["requests"], s["T"], max(s["new"]), max(s["kv"]), s["max_pages"], s["q_start"], s["kv_len"], s["table"])
    need = {"attention": lambda: mdx.paged_attention_workspace(cache, batch), "mass": lambda: mdx.paged_mass_workspace(cache, batch),
            "evict": lambda: mdx.paged_evict_workspace(cache, batch, c["budget"])}.get(c["kind"], lambda: 0)()
    return mdx, cache, batch, torch.zeros(max(need, 16), dtype=torch.uint8, device="cuda")


def run(s):
    c = s["case"]
    if not own:
        if c["kind"] == "attention":
            s["out"], s["lse"] = _attend(s)
            return s["out"], s["lse"]
        return {"append": _append, "mass": _mass, "evict": _evict}[c["kind"]](s)
    if "handles" not in s:
        s["handles"] = _handles(s)
    mdx, cache, batch, ws = s["handles"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["kind"] == "append":
        mdx.paged_append(cache, batch, s["qkv"], s["positions"], s["cos"], s["sin"], s["cos"].shape[0], s["q"], q_norm=s["q_norm"], k_norm=s["k_norm"],
                         eps=EPS, rope_style=c["style"], stream=stream)
        return s["q"], s["k_pages"], s["v_pages"], s["mass"], s["pos"]
    if c["kind"] == "attention":
        mdx.paged_attention(cache, batch, s["q"], s["out"], ws, ws.numel(), lse=s["lse"], scale=s["scale"], stream=stream)
        return s["out"], s["lse"]
    if c["kind"] == "mass":
        mdx.paged_mass(cache, batch, s["q"], s["lse"], ws, ws.numel(), scale=s["scale"], stream=stream)
        return s["mass"]
    mdx.paged_evict(cache, batch, c["budget"], SINK, c["recent"], s["mass_out"], s["pos_out"], ws, ws.numel(), stream=stream)
    return s["k_pages"], s["v_pages"], s["mass_out"], s["pos_out"]


def work(case):
    new, kv = _lengths(case)
    T, nq, nkv, hd = sum(new), case["nq"], case["nkv"], case["hd"]
    seen = sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(new, kv))
    if case["kind"] == "append":
        heads = nq + 2 * nkv
        return dict(bytes=6 * T * heads * hd + 4 * T * hd + 8 * T * nkv, flops=8 * T * (nq + nkv) * hd)
    if case["kind"] == "attention":
        return dict(bytes=4 * sum(kv) * nkv * hd + 4 * T * nq * hd + 4 * T * nq, flops=4 * seen * nq * hd)
    if case["kind"] == "mass":
        return dict(bytes=2 * sum(kv) * nkv * hd + 8 * sum(kv) * nkv + 2 * T * nq * hd + 4 * T * nq, flops=2 * seen * nq * hd)
    b, moved = case["budget"], 0.0
    for L in kv:
        free = b - min(b, SINK + case["recent"])
        moved += 0 if L <= b else (L - b) * b / L if free else L - b
    return dict(bytes=nkv * (sum(8 * L + 8 * min(L, b) for L in kv) + 8 * hd * moved), flops=nkv * sum(kv))


# ---- from the definitions, in 64 bits ---------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    nq, nkv, hd, page = (case[k] for k in ("nq", "nkv", "hd", "page"))
    G, f64 = nq // nkv, torch.float64
    table, starts = s["table"].cpu().numpy(), s["q_start"].cpu().numpy()

    def where(r):
        """Flat (page, row) numbers of request r's cache rows."""
        j = np.arange(s["kv"][r])
        return torch.from_numpy(table[r][j // page].astype(np.int64) * page + j % page).cuda()

    def flat(x):
        """[pages][nkv][page]... as [rows of the pool][nkv]..., a copy."""
        return x.transpose(1, 2).reshape(-1, *x.shape[1:2], *x.shape[3:]).clone()

    def paged(x):
        return x.view(s["pages"], page, *x.shape[1:]).transpose(1, 2).contiguous()

    if case["kind"] == "append":
        x = s["qkv"].to(f64).view(s["T"], -1, hd)
        angles = [s[n].to(f64)[s["positions"].long()].unsqueeze(1) for n in ("cos", "sin")]
        z = torch.complex(*angles)

        def head(x, w):
            if w is not None:
                x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / hd + EPS) * w.to(f64)
            if case["style"] == 0:
                return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], hd // 2, 2).contiguous()) * z).flatten(-2)
            y = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * z
            return torch.cat([y.real, y.imag], -1)

        k, v, mass, pos = flat(s["k_pages"]).to(f64), flat(s["v_pages"]).to(f64), flat(s["mass"]).to(f64), flat(s["pos"])
        q, new_k = head(x[:, :nq], s["q_norm"]), head(x[:, nq:nq + nkv], s["k_norm"])
        for r in range(case["requests"]):
            a, b = int(starts[r]), int(starts[r + 1])
            to = where(r)[s["kv"][r] - (b - a):]
            k[to], v[to], mass[to] = new_k[a:b], x[a:b, nq + nkv:], 0.0
            pos[to] = s["positions"][a:b, None].expand(-1, nkv)
        return q, paged(k), paged(v), paged(mass), paged(pos)

    if case["kind"] in ("attention", "mass"):
        kf, vf = flat(s["k_pages"]), flat(s["v_pages"])
        out = torch.zeros(s["T"], nq, hd, dtype=f64, device="cuda")
        lse = torch.zeros(s["T"], nq, dtype=f64, device="cuda")
        mass = flat(s["mass"]).to(f64) if case["kind"] == "mass" else None
        for r in range(case["requests"]):
            at, L = where(r), s["kv"][r]
            for a in range(int(starts[r]), int(starts[r + 1]), 512):
                b = min(a + 512, int(starts[r + 1]))
                row = L - (int(starts[r + 1]) - torch.arange(a, b, device="cuda"))
                hidden = torch.arange(L, device="cuda")[None] > row[:, None]
                for h in range(nq):
                    w = (s["q"][a:b, h].to(f64) @ kf[at, h // G].to(f64).T) * s["scale"]
                    w = w.masked_fill(hidden, -math.inf)
                    if mass is None:
                        lse[a:b, h] = torch.logsumexp(w, 1)
                        out[a:b, h] = torch.softmax(w, 1) @ vf[at, h // G].to(f64)
                    else:
                        mass[at, h // G] += torch.exp(w - s["lse"][a:b, h, None].to(f64)).sum(0)
        return (out, lse) if mass is None else paged(mass)

    k, v, mass, pos = flat(s["k_pages"]), flat(s["v_pages"]), flat(s["mass"]), flat(s["pos"])
    mass_out, pos_out = torch.zeros_like(mass), torch.zeros_like(pos)
    for r in range(case["requests"]):
        at, L, b = where(r), s["kv"][r], case["budget"]
        m, p = mass[at].cpu().numpy(), pos[at].cpu().numpy()
        first = at[:min(L, b)]
        mass_out[first], pos_out[first] = mass[first], pos[first]
        if L <= b:
            continue
        for h in range(nkv):
            safe = (p[:, h] < SINK) | (p[:, h] > p[:, h].max() - case["recent"])
            stays = np.sort(np.lexsort((np.arange(L), -m[:, h].astype(np.float64), ~safe))[:b])
            gaps, src = np.setdiff1d(np.arange(b), stays), stays[stays >= b]
            gaps, src = at[torch.from_numpy(gaps).cuda()], at[torch.from_numpy(src).cuda()]
            k[gaps, h], v[gaps, h] = k[src, h], v[src, h]
            mass_out[gaps, h], pos_out[gaps, h] = mass[src, h], pos[src, h]
    return paged(k).to(f64), paged(v).to(f64), paged(mass_out).to(f64), paged(pos_out)
