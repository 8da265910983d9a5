"""Arguments that K7 and K8 refuse before any launch (no GPU needed: the C entries check pointers
and sizes on the host, the Python wrappers check tensors)."""

import pytest
import torch

from mdlarc_scale_amd import _lib
from mdlarc_scale_amd import kernels as K

FAKE = 1 << 20                                  # never dereferenced: rejected first
NULL, ALIGN, SHAPE, HEAD, WORKSPACE, DTYPE = -1, -2, -3, -4, -6, -7


@pytest.fixture(scope="module")
def L():
    if not _lib.available():
        pytest.skip("libmdlarc_hip.so not built (python -m mdlarc_scale_amd.build)")
    return _lib.lib()


QK = dict(qkv=FAKE, in_dtype=0, ld=640, rstd=None, pos=FAKE, tab=FAKE, rows=4, row=FAKE, slot=FAKE,
          batch=2, heads=6, kv=2, dim=64, mx=32, my=32, mz=8, px=10, py=10, pz=12, gq=FAKE, gk=FAKE,
          eps=1e-5, scale=1.0, q=FAKE, k=FAKE, v=FAKE, out_dtype=1, slots=16, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(qkv=None), NULL), (dict(pos=None), NULL), (dict(gk=None), NULL), (dict(v=None), NULL),
    (dict(dim=96), HEAD), (dict(in_dtype=2), DTYPE), (dict(out_dtype=-1), DTYPE),
    (dict(heads=5), SHAPE), (dict(kv=0), SHAPE), (dict(ld=636), SHAPE), (dict(pz=13), SHAPE),
    (dict(px=-1, pz=23), SHAPE), (dict(rows=-1), SHAPE), (dict(batch=0), SHAPE),
    (dict(slots=0), SHAPE), (dict(mx=0), SHAPE), (dict(mx=2 ** 31 - 1), SHAPE),
    (dict(rows=2 ** 40), SHAPE), (dict(qkv=FAKE + 8), ALIGN), (dict(ld=642), ALIGN),
    (dict(in_dtype=1, ld=644), ALIGN), (dict(q=FAKE + 4), ALIGN), (dict(gq=FAKE + 4), ALIGN)])
def test_qk_norm_refusals(L, change, code):
    assert L.mdl_qk_norm_rope_cache(*{**QK, **change}.values()) == code


AG = dict(q=FAKE, k=FAKE, v=FAKE, dtype=1, n_seq=2, tokens=9, max_q=5, heads=6, kv=2, dim=64,
          slots=4096, q_offset=FAKE, kv_len=FAKE, causal=1, out=FAKE, form=0, ws=FAKE, ws_bytes=0,
          stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), NULL), (dict(kv_len=None), NULL), (dict(q_offset=None), NULL),
    (dict(out=None), NULL), (dict(dim=80), HEAD), (dict(dtype=3), DTYPE), (dict(heads=7), SHAPE),
    (dict(kv=0), SHAPE), (dict(tokens=-1), SHAPE), (dict(max_q=-2), SHAPE), (dict(form=3), SHAPE),
    (dict(slots=2 ** 31 - 1), SHAPE), (dict(n_seq=2 ** 30 + 1), SHAPE),
    (dict(tokens=2 ** 31 - 1, max_q=2 ** 31 - 1), SHAPE),
    (dict(q=FAKE + 8), ALIGN), (dict(out=FAKE + 2), ALIGN), (dict(ws=FAKE + 4), ALIGN),
    (dict(kv_len=FAKE + 2), ALIGN), (dict(), WORKSPACE)])
def test_grouped_refusals(L, change, code):
    assert L.mdl_attn_grouped(*{**AG, **change}.values()) == code


def test_grouped_workspace(L):
    """Host arithmetic: parts * rows * (dims + 2) floats, none where a launch fills the GPU."""
    few = L.mdl_attn_grouped_workspace_bytes(2, 9, 5, 6, 2, 64, 1, 4096)
    assert few > 0 and few % (9 * 6 * 66 * 4) == 0
    assert L.mdl_attn_grouped_workspace_bytes(64, 6400, 100, 16, 16, 64, 1, 4096) == 0
    assert L.mdl_attn_grouped_workspace_bytes(2, 9, 5, 6, 2, 64, 1, 64) == 0
    assert L.mdl_attn_grouped_workspace_bytes(2, 9, 5, 6, 4, 64, 1, 4096) == 0
    # a bound above the number of rows is that number
    assert (L.mdl_attn_grouped_workspace_bytes(2, 9, 2 ** 31 - 1, 6, 2, 64, 1, 4096) ==
            L.mdl_attn_grouped_workspace_bytes(2, 9, 9, 6, 2, 64, 1, 4096) > 0)


SH = dict(q=FAKE, pk=FAKE, pv=FAKE, row_offset=FAKE, prefix_len=FAKE, n_prefix=1, prefix_slots=512,
          max_rows=4, k=FAKE, v=FAKE, kv_len=FAKE, batch=4, slots=64, dtype=1, heads=6, kv=2, dim=64,
          out=FAKE, form=0, ws=FAKE, ws_bytes=0, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(pk=None), NULL), (dict(row_offset=None), NULL), (dict(ws=None), NULL),
    (dict(dim=32), HEAD), (dict(dtype=2), DTYPE), (dict(kv=4), SHAPE), (dict(n_prefix=0), SHAPE),
    (dict(max_rows=0), SHAPE), (dict(batch=-1), SHAPE), (dict(prefix_slots=-1), SHAPE),
    (dict(form=-1), SHAPE), (dict(pv=FAKE + 8), ALIGN), (dict(prefix_len=FAKE + 1), ALIGN),
    (dict(), WORKSPACE)])
def test_shared_refusals(L, change, code):
    assert L.mdl_attn_decode_shared(*{**SH, **change}.values()) == code


def test_wrappers_refuse_host_tensors_and_shapes():
    q, c = torch.zeros(4, 6, 64), torch.zeros(2, 2, 8, 64)
    off, n = torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        K.attn_grouped(q, c, c, off, n, 2, torch.zeros_like(q))
    with pytest.raises(ValueError, match="64 or 128"):
        K.attn_grouped(q[:, :, :32], c, c, off, n, 2, q)
    with pytest.raises(ValueError, match="64 or 128"):
        K.attn_decode_shared(q[0], c, c, off, n, 2, c, c, n, q, q)
    with pytest.raises(ValueError, match="do not hold"):
        K.qk_norm_rope_cache(torch.zeros(3, 448), None, off, q, (8, 8, 8, 10, 10, 12), q, q, 1e-5,
                             off, off, 1.0, q, c, c)
    with pytest.raises(ValueError, match="64 or 128"):
        K.qk_norm_rope_cache(torch.zeros(3, 640), None, off, q, (8, 8, 8, 10, 10, 12), q, q, 1e-5,
                             off, off, 1.0, q, c[..., :48], c)
    with pytest.raises(ValueError, match="GPU tensor"):
        K.qk_norm_rope_cache(torch.zeros(3, 640), None, off, q, (8, 8, 8, 10, 10, 12), q, q, 1e-5,
                             off, off, 1.0, q, c, c)


@pytest.mark.parametrize("most", [2 ** 31, 2 ** 32, 2 ** 32 + 1, 2 ** 40])
def test_bounds_above_the_rows_count_as_the_rows(L, most):
    """max_q and max_rows are bounds: one that a C int does not hold is still one, no small number
    or zero (for which the entries have nothing to do)."""
    q, cache = torch.zeros(9, 6, 64), torch.zeros(2, 2, 4096, 64)
    assert K.attn_grouped_workspace_bytes(q, cache, most) == \
        K.attn_grouped_workspace_bytes(q, cache, 9) > 0
    own = torch.zeros(9, 2, 16, 64)
    assert K.attn_decode_shared_workspace_bytes(q, cache, own, most) == \
        K.attn_decode_shared_workspace_bytes(q, cache, own, 9) > 0


@pytest.mark.parametrize("most", [-1, -2 ** 31, -2 ** 32, -2 ** 32 + 5])
def test_bounds_below_zero_need_no_workspace(L, most):
    q, cache = torch.zeros(9, 6, 64), torch.zeros(2, 2, 4096, 64)
    assert K.attn_grouped_workspace_bytes(q, cache, most) == 0
    assert K.attn_decode_shared_workspace_bytes(q, cache, torch.zeros(9, 2, 16, 64), most) == 0


def test_qk_norm_refuses_a_cache_without_rows():
    """q_out is written for every token, whether its slot is in the cache or not, so the wrapper does
    not pass over tokens that no cache row can hold."""
    qkv, none = torch.zeros(3, 8 * 64), torch.zeros(0, 2, 8, 64)
    off, gain = torch.zeros(3, dtype=torch.int32), torch.ones(64)
    with pytest.raises(ValueError, match="batch 0"):
        K.qk_norm_rope_cache(qkv, None, off, gain, (8, 8, 8, 10, 10, 12), gain, gain, 1e-5, off, off,
                             1.0, torch.zeros(3, 4, 64), none, none)


@pytest.mark.parametrize("most", [5, 2 ** 20, 2 ** 31 - 1])
def test_shared_bound_above_the_rows_is_their_number(L, most):
    """The entry takes every bound that its workspace function does (and stops at a workspace of 0
    bytes here); the refusals of a batch below zero or a bound of none stay."""
    need = L.mdl_attn_decode_shared_workspace_bytes
    assert need(4, 1, most, 6, 2, 64, 1, 512, 64) == need(4, 1, 4, 6, 2, 64, 1, 512, 64) > 0
    call = L.mdl_attn_decode_shared
    assert call(*{**SH, "max_rows": most}.values()) == WORKSPACE
    assert call(*{**SH, "max_rows": most, "batch": 0}.values()) == 0
    assert call(*{**SH, "max_rows": most, "batch": -1}.values()) == SHAPE
    assert call(*{**SH, "max_rows": 0, "batch": 0}.values()) == SHAPE
    assert call(*{**SH, "max_rows": -1}.values()) == SHAPE


@pytest.mark.parametrize("geom,sent", [
    ((2 ** 32 + 32, 1, 1, 1, 31, 0), (2 ** 31 - 1, 1, 1, 1, 31, 0)),
    ((1, -2 ** 32 + 32, 1, 0, 32, 0), (1, -1, 1, 0, 32, 0)),
    ((32, 32, 8, -2 ** 32 + 10, 10, 12), (32, 32, 8, -1, 10, 12)),
    ((32, 32, 8, 10, 2 ** 32 + 10, 12), (32, 32, 8, 10, 2 ** 31 - 1, 12))])
def test_axes_that_a_c_int_does_not_hold_are_refused(L, monkeypatch, geom, sent):
    """They reach the entry as numbers that it refuses, not as their low 32 bits, for which the table
    was not checked."""
    got = []
    monkeypatch.setattr(K, "_need_all", lambda dev, specs: None)
    monkeypatch.setattr(K, "_launch", lambda dev, name, *args: got.append(args))
    n, gain = torch.zeros(3, dtype=torch.int32), torch.ones(64)
    cache = torch.zeros(2, 2, 8, 64)
    K.qk_norm_rope_cache(torch.zeros(3, 8 * 64), None, n, gain, geom, gain, gain, 1e-5, n, n, 1.0,
                         torch.zeros(3, 4, 64), cache, cache)
    at = list(QK).index("mx") - list(QK).index("in_dtype") + 1
    assert got[0][at:at + 6] == sent
    fake = {**QK, **dict(zip(("mx", "my", "mz", "px", "py", "pz"), sent))}
    assert L.mdl_qk_norm_rope_cache(*fake.values()) == SHAPE
