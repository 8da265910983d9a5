"""Sizes whose launch would count 2^32 threads or more are refused before any launch (no GPU needed): a
grid counts its threads in 32 bits, and one with more is cut without an error."""

import pytest

from mdlarc_scale_amd import _lib

from .test_grouped_refusals import AG, QK, SH
from .test_paged_refusals import AP, AT, RO

FAKE, SHAPE = 1 << 20, -3


@pytest.fixture(scope="module")
def L():
    if not _lib.available():
        pytest.skip("libmdlarc_hip.so not built (python -m mdlarc_scale_amd.build)")
    return _lib.lib()


ROPE = [FAKE, 768, FAKE, FAKE, FAKE]     # qkv, ld, rstd, pos, table


@pytest.mark.parametrize("name,args", [
    # caches in pages and grouped heads: a wave takes three passes of a token, a block a pair's tile
    ("mdl_rope_cache_paged", {**AP, "rows": 2 ** 27}.values()),
    ("mdl_paged_rows", {**RO, "n_seq": 2 ** 24}.values()),
    ("mdl_attn_paged", {**AT, "n_seq": 2 ** 24, "tokens": 2 ** 24, "max_q": 1, "ws": None}.values()),
    ("mdl_attn_paged", {**AT, "n_seq": 2 ** 23, "tokens": 2 ** 23, "max_q": 1, "ws": None,
                        "page_dtype": 2, "ks": FAKE, "vs": FAKE}.values()),
    # one token of many: the merge's rows
    ("mdl_attn_paged", {**AT, "n_seq": 1, "tokens": 2 ** 25, "max_q": 1, "ws_bytes": 2 ** 62}.values()),
    ("mdl_attn_grouped", {**AG, "n_seq": 1, "tokens": 2 ** 25, "max_q": 1,
                          "ws_bytes": 2 ** 62}.values()),
    ("mdl_attn_grouped", {**AG, "n_seq": 2 ** 24, "tokens": 2 ** 24, "max_q": 1, "ws": None}.values()),
    ("mdl_attn_decode_shared", {**SH, "batch": 2 ** 25, "ws_bytes": 2 ** 62}.values()),
    ("mdl_qk_norm_rope_cache", {**QK, "rows": 2 ** 27}.values()),
    # a wave or a block a row, sixteen rows or a stretch of channels
    ("mdl_embed_rmsnorm", [FAKE, None, FAKE, None, 0, 14, 0, 2 ** 27, 1, 256, FAKE, 1e-5, FAKE, FAKE,
                           FAKE, 0, None]),
    ("mdl_embed_rmsnorm_bf16", [FAKE, None, FAKE, None, 14, 0, 2 ** 28, 1, 256, FAKE, 1e-5, FAKE, FAKE,
                                None]),
    ("mdl_decode_embed", [FAKE, None, FAKE, None, 0, 14, 0, 2 ** 27, 256, FAKE, 1e-5, FAKE, FAKE, FAKE,
                          30, 30, FAKE, None, FAKE, FAKE, FAKE, 0, None]),
    ("mdl_add_rmsnorm", [FAKE, FAKE, None, 2 ** 27, 256, FAKE, 1e-5, FAKE, FAKE, 0, None]),
    ("mdl_qkv_rope_cache", [*ROPE, 2 ** 27, 1, 4, 64, 32, 32, 8, 10, 10, 12, 1.0, FAKE, FAKE, FAKE, 1,
                            4, 0, None, None]),
    ("mdl_swiglu", [FAKE, 4096, None, None, None, 2 ** 26, 2048, FAKE, 0, None]),
    ("mdl_swiglu_bf16", [FAKE, 4096, None, None, None, 2 ** 27, 2048, FAKE, None]),
    ("mdl_tile_matrix", [FAKE, 2048, 2 ** 26, 2048, FAKE, None]),
    ("mdl_zero_tiled_rows", [FAKE, 0, 2 ** 26, 2048, None]),
    ("mdl_lm_head", [FAKE, None, 2 ** 25, 256, FAKE, 1e-5, FAKE, 14, FAKE, FAKE, None, 0, None]),
    ("mdl_grid_init", [FAKE, FAKE, None, None, 2 ** 27, 1, 30, 30, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE,
                       None]),
    ("mdl_attn_decode", [FAKE, FAKE, FAKE, 2 ** 23, 4, 64, 16, None, 0, None, None, None, 3, None, None,
                         0, 2 ** 20, FAKE, 0, None]),
])
def test_grids_of_too_many_threads_are_refused(L, name, args):
    assert getattr(L, name)(*args) == SHAPE
