"""Arguments that K9, K10 and K11 refuse before any launch (no GPU needed), and the plain forms that
their GPU tests go by."""

import pytest
import torch

from mdlarc_scale_amd import _lib
from mdlarc_scale_amd import kernels as K

from .paged_ref import from_fp4, kept_tokens, sampled, to_fp4

FAKE = 1 << 20                                  # never dereferenced: rejected first
NULL, ALIGN, SHAPE, HEAD, WORKSPACE, DTYPE = -1, -2, -3, -4, -6, -7
F32, BF, U8, I32 = torch.float32, torch.bfloat16, torch.uint8, torch.int32


@pytest.fixture(scope="module")
def L():
    if not _lib.available():
        pytest.skip("libmdlarc_hip.so not built (python -m mdlarc_scale_amd.build)")
    return _lib.lib()


AP = dict(qkv=FAKE, in_dtype=0, ld=640, rstd=None, pos=FAKE, tab=FAKE, rows=4, row=FAKE, slot=FAKE,
          table=FAKE, table_ld=3, n_seq=2, width=3, n_pages=7, page=16, heads=6, kv=2, dim=64, mx=32,
          my=32, mz=8, px=10, py=10, pz=12, gq=None, gk=None, eps=1e-5, scale=1.0, q=FAKE, q_dtype=1,
          k=FAKE, v=FAKE, page_dtype=1, ks=None, vs=None, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(qkv=None), NULL), (dict(table=None), NULL), (dict(v=None), NULL), (dict(gq=FAKE), NULL),
    (dict(page_dtype=2), NULL), (dict(page_dtype=2, ks=FAKE), NULL), (dict(dim=96), HEAD),
    (dict(in_dtype=2), DTYPE), (dict(q_dtype=0), DTYPE), (dict(q_dtype=2, page_dtype=2, ks=FAKE,
                                                               vs=FAKE), DTYPE),
    (dict(page_dtype=3), DTYPE), (dict(heads=5), SHAPE), (dict(kv=0), SHAPE), (dict(ld=636), SHAPE),
    (dict(pz=13), SHAPE), (dict(rows=-1), SHAPE), (dict(page=8), SHAPE), (dict(page=24), SHAPE),
    (dict(page=8192), SHAPE), (dict(n_pages=0), SHAPE), (dict(table_ld=2), SHAPE),
    (dict(width=2 ** 27, table_ld=2 ** 27), SHAPE), (dict(mx=0), SHAPE), (dict(mx=2 ** 31 - 1), SHAPE),
    (dict(rows=2 ** 40), SHAPE), (dict(n_seq=-1), SHAPE), (dict(qkv=FAKE + 8), ALIGN),
    (dict(ld=642), ALIGN), (dict(in_dtype=1, ld=644), ALIGN), (dict(k=FAKE + 4), ALIGN),
    (dict(table=FAKE + 2), ALIGN), (dict(gq=FAKE + 4, gk=FAKE), ALIGN)])
def test_append_refusals(L, change, code):
    assert L.mdl_rope_cache_paged(*{**AP, **change}.values()) == code


RO = dict(k=FAKE, v=FAKE, page_dtype=1, ks=None, vs=None, table=FAKE, table_ld=3, n_seq=2, width=3,
          n_pages=7, page=16, kv=2, dim=64, start=FAKE, count=FAKE, run=5, ko=FAKE, vo=FAKE,
          out_dtype=1, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(k=None), NULL), (dict(count=None), NULL), (dict(page_dtype=2), NULL), (dict(dim=80), HEAD),
    (dict(out_dtype=0), DTYPE), (dict(page_dtype=2, ks=FAKE, vs=FAKE, out_dtype=2), DTYPE),
    (dict(run=-1), SHAPE), (dict(run=2 ** 31 - 1), SHAPE), (dict(page=17), SHAPE),
    (dict(n_pages=-1), SHAPE), (dict(kv=0), SHAPE), (dict(n_seq=2 ** 30, run=4096, kv=9), SHAPE),
    (dict(ko=FAKE + 8), ALIGN), (dict(start=FAKE + 1), ALIGN)])
def test_rows_refusals(L, change, code):
    assert L.mdl_paged_rows(*{**RO, **change}.values()) == code


AT = dict(q=FAKE, dtype=1, k=FAKE, v=FAKE, page_dtype=1, ks=None, vs=None, n_pages=600, page=16,
          table=FAKE, table_ld=256, width=256, n_seq=2, tokens=9, max_q=5, heads=6, kv=2, dim=64,
          q_offset=FAKE, kv_len=FAKE, causal=1, out=FAKE, form=0, ws=FAKE, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), NULL), (dict(table=None), NULL), (dict(out=None), NULL),
    (dict(page_dtype=2, ks=FAKE), NULL), (dict(dim=80), HEAD), (dict(dtype=3), DTYPE),
    (dict(dtype=2), DTYPE), (dict(page_dtype=0), DTYPE), (dict(heads=7), SHAPE), (dict(kv=0), SHAPE),
    (dict(tokens=-1), SHAPE), (dict(max_q=-2), SHAPE), (dict(form=3), SHAPE), (dict(page=40), SHAPE),
    (dict(width=2 ** 27, table_ld=2 ** 27), SHAPE), (dict(table_ld=255), SHAPE),
    (dict(n_pages=0), SHAPE), (dict(n_seq=2 ** 30 + 1), SHAPE),
    (dict(tokens=2 ** 31 - 1, max_q=2 ** 31 - 1), SHAPE), (dict(q=FAKE + 8), ALIGN),
    (dict(ws=FAKE + 4), ALIGN), (dict(table=FAKE + 2), ALIGN), (dict(), WORKSPACE)])
def test_attention_refusals(L, change, code):
    assert L.mdl_attn_paged(*{**AT, **change}.values()) == code


def test_attention_workspace(L):
    """That of the contiguous form with as many slots."""
    need = L.mdl_attn_paged_workspace_bytes
    assert need(2, 9, 5, 6, 2, 64, 1, 1, 256, 16) == \
        L.mdl_attn_grouped_workspace_bytes(2, 9, 5, 6, 2, 64, 1, 4096) > 0
    assert need(2, 9, 5, 6, 2, 64, 1, 2, 256, 16) > 0
    assert need(2, 9, 5, 6, 2, 64, 1, 0, 256, 16) == 0      # refused types and sizes
    assert need(2, 9, 5, 6, 2, 64, 1, 1, 256, 8) == 0
    assert need(64, 6400, 100, 16, 16, 64, 1, 1, 256, 16) == 0


SA = dict(logits=FAKE, dtype=0, ld=100, rows=4, vocab=100, u=FAKE, t=None, k=None, p=None, m=None,
          token=FAKE, logprob=None, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(logits=None), NULL), (dict(u=None), NULL), (dict(token=None), NULL), (dict(dtype=2), DTYPE),
    (dict(rows=-1), SHAPE), (dict(vocab=0), SHAPE), (dict(ld=99), SHAPE),
    (dict(vocab=2 ** 20 + 1, ld=2 ** 21), SHAPE), (dict(logits=FAKE + 2), ALIGN),
    (dict(dtype=1, logits=FAKE + 1), ALIGN), (dict(token=FAKE + 4), ALIGN), (dict(k=FAKE + 2), ALIGN),
    (dict(ws=FAKE + 4), ALIGN), (dict(vocab=5000, ld=5000), WORKSPACE),
    (dict(vocab=5000, ld=5000, ws=FAKE, ws_bytes=100), WORKSPACE),
    (dict(vocab=5000, ld=5000, ws=FAKE, rows=2 ** 31 - 1), SHAPE)])
def test_sample_refusals(L, change, code):
    assert L.mdl_sample_tokens(*{**SA, **change}.values()) == code


def test_sample_workspace(L):
    need = L.mdl_sample_workspace_bytes
    assert need(64, 4096) == need(0, 9000) == need(5, 2 ** 20 + 1) == 0
    assert need(1, 4097) > 0 and need(64, 2 ** 20) >= 64 * 64 * 8192
    assert K.sample_workspace_bytes(3, 10 ** 5) == need(3, 10 ** 5)


def test_empty_calls_have_nothing_to_do(L):
    assert L.mdl_rope_cache_paged(*{**AP, "rows": 0}.values()) == 0
    assert L.mdl_paged_rows(*{**RO, "run": 0}.values()) == 0
    assert L.mdl_paged_rows(*{**RO, "n_seq": 0}.values()) == 0
    assert L.mdl_attn_paged(*{**AT, "tokens": 0}.values()) == 0
    assert L.mdl_sample_tokens(*{**SA, "rows": 0}.values()) == 0


def test_wrappers_refuse():
    k, s = torch.zeros(3, 2, 16, 64), torch.zeros(3, 2, 16, 2, dtype=U8)
    k4 = torch.zeros(3, 2, 16, 32, dtype=U8)
    table, n = torch.zeros(2, 4, dtype=I32), torch.zeros(2, dtype=I32)
    q, off = torch.zeros(4, 6, 64), torch.zeros(3, dtype=I32)

    def attend(q=q, k=k, v=k, table=table, off=off, n=n, **kw):
        K.attn_paged(q, k, v, table, off, n, 2, torch.zeros_like(q), **kw)
    for what, call in [
            ("GPU tensor", lambda: attend()),
            ("both be", lambda: attend(v=k[:2])),
            ("head_dim of 64", lambda: attend(k=k[..., :48], v=k[..., :48])),
            ("multiples of 16", lambda: attend(k=k[:, :, :8], v=k[:, :, :8])),
            ("needs pages", lambda: attend(k=k[:0], v=k[:0])),
            ("sequences, pages", lambda: attend(table=n)),
            ("int32", lambda: attend(table=table.long())),
            ("contiguous rows", lambda: attend(table=table[:, ::2])),
            ("do not overlap", lambda: attend(table=table[:1].expand(2, -1))),
            ("no columns", lambda: attend(table=table[:, :0])),
            ("only 4-bit", lambda: attend(k_scale=s, v_scale=s)),
            ("k_scale must", lambda: attend(k=k4, v=k4)),
            ("v_scale must", lambda: attend(k=k4, v=k4, k_scale=s, v_scale=s[:2])),
            ("multiple of 2 heads", lambda: attend(q=q[:, :5])),
            ("must have 3 and 2", lambda: attend(n=off)),
            ("GPU tensor", lambda: K.paged_rows(k, k, table, n, n, torch.zeros(2, 2, 3, 64),
                                                torch.zeros(2, 2, 3, 64))),
            ("both be", lambda: K.paged_rows(k, k, table, n, n, torch.zeros(2, 2, 3, 64),
                                             torch.zeros(2, 2, 4, 64))),
            ("elements", lambda: K.paged_rows(k, k, table, off, n, torch.zeros(2, 2, 3, 64),
                                              torch.zeros(2, 2, 3, 64))),
            ("logits must", lambda: K.sample_tokens(torch.zeros(3), n, n)),
            ("rows of logits", lambda: K.sample_tokens(torch.zeros(4, 8)[:, ::2], n, n)),
            ("bfloat16 or float32", lambda: K.sample_tokens(torch.zeros(4, 8).half(), n, n)),
            ("GPU tensors", lambda: K.sample_tokens(torch.zeros(4, 8), n, n))]:
        with pytest.raises(ValueError, match=what):
            call()
    geom, ones = (8, 8, 8, 10, 10, 12), torch.ones(64)

    def append(qkv=torch.zeros(3, 640), geom=geom, **kw):
        K.rope_cache_paged(qkv, None, off, ones, geom, off, off, table, 1.0, torch.zeros(3, 6, 64), k,
                           k, **kw)
    for what, call in [("GPU tensor", lambda: append()),
                       ("do not hold", lambda: append(torch.zeros(3, 448))),
                       ("must be contiguous", lambda: append(torch.zeros(3, 1280)[:, ::2])),
                       ("together", lambda: append(q_gamma=ones)),
                       ("out of range", lambda: append(geom=(2 ** 31, 8, 8, 10, 10, 12))),
                       ("out of range", lambda: append(geom=(8, 8, 8, -1, 21, 12)))]:
        with pytest.raises(ValueError, match=what):
            call()


@pytest.mark.parametrize("most", [2 ** 31, 2 ** 32 + 1, 2 ** 40])
def test_bounds_above_the_rows_count_as_the_rows(L, most):
    q, k, table = torch.zeros(9, 6, 64), torch.zeros(3, 2, 16, 64), torch.zeros(2, 256, dtype=I32)
    need = K.attn_paged_workspace_bytes
    assert need(q, k, table, most) == need(q, k, table, 9) > 0
    assert need(q, k, table, -most) == 0


# ---- the plain forms ---------------------------------------------------------------------------

def test_plain_fp4():
    x = torch.tensor([7.0, 6.99, -6.5, 5.0, 5.01, 3.5, 2.5, 0.25, 0.26, -0.75] + [0.0] * 22)
    codes, scale = to_fp4(torch.stack([x, x * 0.99, x * 0]))
    assert scale[:, 0].tolist() == [128, 127, 27]
    assert from_fp4(codes, scale)[1, :10].tolist() == [6, 6, -6, 4, 4, 3, 2, 0, 0.5, -0.5]
    assert from_fp4(codes, scale)[0, :6].tolist() == [8, 6, -6, 4, 6, 4]
    # within half a step everywhere: the largest error is a third of a number's size, or 1/4
    y = torch.randn(50, 64, generator=torch.Generator().manual_seed(1))
    c, s = to_fp4(y)
    power = torch.pow(2.0, s.double() - 127).repeat_interleave(32, -1)
    err = (from_fp4(c, s) - y.double()).abs() / power
    size = y.double().abs() / power
    assert bool((err <= torch.where(size < 2, 0.25, torch.where(size < 4, 0.5, 1.0))).all())


def test_plain_order():
    x = torch.tensor([1.0, 3.0, 3.0, -float("inf"), float("nan"), 2.0])
    assert kept_tokens(x, top_k=2)[0].tolist() == [1, 2]
    assert kept_tokens(x, top_p=0.3)[0].tolist() == [1]
    assert sampled(x, 0.0)[0] == 0 and sampled(x, 1 - 2.0 ** -24)[0] == 5
    assert sampled(x, 0.5, temperature=0.0)[:2] == (1, 0.0)


@pytest.mark.parametrize("name,plain,refusals", [
    ("mdl_rope_cache_paged", AP, test_append_refusals), ("mdl_paged_rows", RO, test_rows_refusals),
    ("mdl_attn_paged", AT, test_attention_refusals), ("mdl_sample_tokens", SA, test_sample_refusals)])
def test_blocks_hold_the_arguments(L, name, plain, refusals):
    """The forms with their arguments in a block refuse what the plain ones do."""
    entry, pack = _lib.BLOCKS[name]
    for change, code in refusals.pytestmark[0].args[1]:
        values = list({**plain, **change}.values())[:-1]
        assert getattr(L, entry)(pack(*(0 if v is None else v for v in values)), None) == code, change
    assert getattr(L, entry)(None, None) == NULL
