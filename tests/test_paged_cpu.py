"""The paged cache's entry points refuse bad arguments before anything reaches a
device, say why, and take empty batches."""
import ctypes as C

import numpy as np
import pytest

import paged64

A = 4096        # an aligned address that is never read


def _cache(mdx, **over):
    f = dict(dtype="fp16", num_q_heads=4, num_kv_heads=2, head_dim=64, page_size=16, n_pages=8, k_pages=A, v_pages=A, mass=A, pos=A)
    f.update(over)
    return mdx.paged_cache(**f)


def _batch(mdx, **over):
    f = dict(n_req=2, n_tokens=3, max_q_len=2, max_kv_len=40, max_pages=3, q_start=A, kv_len=A, block_table=A)
    f.update(over)
    return mdx.paged_batch(**f)


CALLS = {
    "append": lambda m, c, b, **k: m.paged_append(c, b, **{**dict(qkv=A, positions=A, cos=A, sin=A, max_pos=64, q_out=A), **k}),
    "attention": lambda m, c, b, **k: m.paged_attention(c, b, **{**dict(q=A, out=2 * A, workspace=A, workspace_bytes=1 << 40), **k}),
    "mass": lambda m, c, b, **k: m.paged_mass(c, b, **{**dict(q=A, lse=A, workspace=A, workspace_bytes=1 << 40), **k}),
    "evict": lambda m, c, b, **k: m.paged_evict(c, b, **{**dict(budget=8, sink=2, recent=4, mass_out=A, pos_out=A, workspace=A, workspace_bytes=1 << 40), **k}),
}


def _refused(mdx, call, c, b, rc, says, **k):
    with pytest.raises(RuntimeError) as e:
        CALLS[call](mdx, c, b, **k)
    assert f"({rc})" in str(e.value) and says in str(e.value), str(e.value)


@pytest.mark.parametrize("call", list(CALLS))
@pytest.mark.parametrize("over,rc,says", [
    (dict(dtype=2), -1, "unknown type"), (dict(dtype=-1), -1, "unknown type"),
    (dict(num_q_heads=5), -1, "multiple of num_kv_heads"), (dict(num_kv_heads=0), -1, "multiple of num_kv_heads"),
    (dict(num_q_heads=0), -1, "multiple of num_kv_heads"), (dict(num_q_heads=16386), -1, "too many heads"),
    (dict(head_dim=96), -5, "head_dim"), (dict(head_dim=0), -5, "head_dim"),
    (dict(page_size=8), -5, "page_size"), (dict(page_size=24), -5, "page_size"), (dict(page_size=2048), -5, "page_size"),
    (dict(page_size=0), -5, "page_size"), (dict(page_size=-16), -5, "page_size"),
    (dict(n_pages=0), -1, "no pages"), (dict(k_pages=None), -1, "no pages"), (dict(v_pages=None), -1, "no pages"),
    (dict(k_pages=A + 8), -1, "16-byte aligned"), (dict(v_pages=A + 2), -1, "16-byte aligned"), (dict(mass=A + 4), -1, "16-byte aligned"),
    (dict(pos=A + 8), -1, "16-byte aligned"),
])
def test_refused_caches(mdx, call, over, rc, says):
    _refused(mdx, call, _cache(mdx, **over), _batch(mdx), rc, says)


@pytest.mark.parametrize("call", list(CALLS))
@pytest.mark.parametrize("over,says", [
    (dict(n_req=-1), "n_req"), (dict(n_req=65536), "n_req"), (dict(max_kv_len=-1), "negative"), (dict(max_pages=-1), "negative"),
    (dict(kv_len=None), "no kv_len"), (dict(block_table=None), "no kv_len or block_table"), (dict(kv_len=A + 1), "4-byte aligned"),
])
def test_refused_batches(mdx, call, over, says):
    _refused(mdx, call, _cache(mdx), _batch(mdx, **over), -1, says)


@pytest.mark.parametrize("call", ["append", "attention", "mass"])
@pytest.mark.parametrize("over,says", [(dict(n_tokens=-1), "negative n_tokens"), (dict(max_q_len=-1), "negative"), (dict(q_start=None), "no q_start")])
def test_refused_rows_of_a_batch(mdx, call, over, says):
    _refused(mdx, call, _cache(mdx), _batch(mdx, **over), -1, says)


@pytest.mark.parametrize("call,over,says", [
    ("append", dict(qkv=None), "qkv"), ("append", dict(qkv=A + 4), "qkv"), ("append", dict(qkv_stride=511), "qkv_stride"),
    ("append", dict(qkv_stride=514), "qkv_stride"), ("append", dict(positions=None), "positions"), ("append", dict(cos=None), "tables"),
    ("append", dict(sin=A + 4), "tables"), ("append", dict(q_norm=A + 4), "norms"), ("append", dict(max_pos=0), "max_pos"),
    ("append", dict(rope_style=2), "rope_style"), ("append", dict(eps=-1e-6), "eps"), ("append", dict(eps=float("nan")), "eps"),
    ("append", dict(q_out=None), "no q_out"), ("append", dict(q_out=A + 2), "aligned"), ("append", dict(q_stride=248), "stride"),
    ("append", dict(q_stride=260), "stride"),
    ("attention", dict(q=None), "no q"), ("attention", dict(q=A + 2), "aligned"), ("attention", dict(out=None), "no out"),
    ("attention", dict(q_stride=255), "stride"), ("attention", dict(out_stride=257), "stride"), ("attention", dict(scale=-1.0), "scale"),
    ("attention", dict(scale=float("nan")), "scale"), ("attention", dict(scale=1e-39), "scale"), ("attention", dict(scale=2e30), "scale"),
    ("attention", dict(q=A, out=A), "apart"), ("attention", dict(scale=float("inf")), "scale"), ("attention", dict(lse=A + 1), "lse"),
    ("mass", dict(q=None), "no q"), ("mass", dict(lse=None), "lse"), ("mass", dict(q_stride=0), "stride"), ("mass", dict(scale=-0.5), "scale"),
    ("evict", dict(budget=-1), "budget"), ("evict", dict(sink=-1), "budget"), ("evict", dict(recent=-1), "budget"),
    ("evict", dict(sink=5), "budget"), ("evict", dict(recent=2 ** 31 - 1), "budget"), ("evict", dict(mass_out=None), "mass_out"),
    ("evict", dict(pos_out=None), "mass_out"), ("evict", dict(workspace_bytes=0), "workspace"), ("evict", dict(workspace=None), "workspace"),
    ("evict", dict(workspace=A + 4), "workspace"),
])
def test_refused_arguments(mdx, call, over, says):
    _refused(mdx, call, _cache(mdx), _batch(mdx), -1, says, **over)


@pytest.mark.parametrize("call", list(CALLS))
def test_refused_caches_beyond_32_bit_rows(mdx, call):
    """More rows than kernels count; either bound on its own may be larger."""
    big = _batch(mdx, max_kv_len=2 ** 31 - 1, max_pages=2 ** 29 // 16 + 1)
    _refused(mdx, call, _cache(mdx), big, -1, "2^29")
    assert mdx.paged_attention_workspace(_cache(mdx), big) == 0
    for k in (dict(max_kv_len=2 ** 31 - 1, max_pages=2 ** 29 // 16), dict(max_kv_len=2 ** 29, max_pages=2 ** 31 - 1)):
        assert 0 < mdx.paged_attention_workspace(_cache(mdx), _batch(mdx, **k)) < 1 << 40


def test_refused_without_mass_or_pos(mdx):
    _refused(mdx, "mass", _cache(mdx, mass=None), _batch(mdx), -1, "keeps no mass")
    _refused(mdx, "evict", _cache(mdx, mass=None), _batch(mdx), -1, "no mass or no pos")
    _refused(mdx, "evict", _cache(mdx, pos=None), _batch(mdx), -1, "no mass or no pos")


def test_refused_workspaces(mdx):
    """A split attention needs its workspace, whole and aligned."""
    c, b = _cache(mdx), _batch(mdx, max_kv_len=4096, max_pages=256)
    need = mdx.paged_attention_workspace(c, b)
    assert need > 0
    for k in (dict(workspace_bytes=need - 1), dict(workspace=None, workspace_bytes=need), dict(workspace=A + 8, workspace_bytes=need)):
        _refused(mdx, "attention", c, b, -1, "workspace", **k)


@pytest.mark.parametrize("call", list(CALLS))
def test_null_structs_are_refused(mdx, call):
    L, p = mdx.lib(), C.c_void_p(A)
    fn = {"append": lambda c, b: L.mdx_paged_append(c, b, p, 512, p, None, None, 1e-6, p, p, 64, 0, p, 256, None),
          "attention": lambda c, b: L.mdx_paged_attention(c, b, p, 256, 0.0, C.c_void_p(2 * A), 256, None, p, 1 << 40, None),
          "mass": lambda c, b: L.mdx_paged_mass(c, b, p, 256, 0.0, p, p, 1 << 40, None),
          "evict": lambda c, b: L.mdx_paged_evict(c, b, 8, 2, 4, p, p, p, 1 << 40, None)}[call]
    assert fn(None, _batch(mdx)) == -1 and fn(_cache(mdx), None) == -1
    assert L.mdx_paged_attention_workspace(None, _batch(mdx)) == 0 and L.mdx_paged_evict_workspace(_cache(mdx), None, 8) == 0


@pytest.mark.parametrize("call", list(CALLS))
def test_empty_batches_are_taken(mdx, call):
    """No requests: nothing is launched, on a machine without a GPU too."""
    CALLS[call](mdx, _cache(mdx), _batch(mdx, n_req=0, q_start=None, kv_len=None, block_table=None))
    if call != "evict":
        CALLS[call](mdx, _cache(mdx), _batch(mdx, n_tokens=0))


def test_reference_rounding():
    """The tests' own conversion to bf16 rounds to nearest even."""
    x = np.array([1.0, 1 + 2 ** -8, 1 + 3 * 2 ** -8, -1 - 2 ** -8 - 2 ** -20, 3e38, np.inf, 0.0], np.float32)
    got = paged64.wide(paged64.to16(x, "bf16"), "bf16")
    assert np.array_equal(got[:4], [1.0, 1.0, 1 + 2 ** -6, -1 - 2 ** -7]) and np.isinf(got[5]) and got[6] == 0
