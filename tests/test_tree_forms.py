"""Which kernel and which cut a call of tree attention gets, decided on the host (no GPU): the forms that the GPU tests
mean to run are the ones their sizes choose."""
import ctypes

import pytest
import torch

from xllm_wxh_amd import _lib, ops
from xllm_wxh_amd import build as xbuild

FORMS = ops.TREE_DESCRIBE_FIELDS


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        xbuild.build_library(verbose=False)
    return _lib.load()


def describe(lib, batch, n, hq, hkv, D, bs, kv=_lib.BF16, q=_lib.BF16, hints=(0, 0), status=_lib.OK, **cache):
    d, a = _lib.KvCacheDesc(), _lib.DecodeArgs()
    d.k_cache, d.v_cache, d.k_scale, d.v_scale = 0x10000, 0x20000, 0x30000, 0x40000
    d.num_blocks, d.block_size, d.num_kv_heads, d.head_dim, d.dtype = 1000, bs, hkv, D, kv
    d.stride_block, d.stride_head, d.stride_slot = hkv * bs * D, bs * D, D
    d.scale_stride_block, d.scale_stride_head, d.scale_stride_slot = hkv * bs, bs, 1
    for name, value in cache.items():
        setattr(d, name, value)
    a.q, a.out, a.block_table, a.seq_lens = 0x50000, 0x60000, 0x70000, 0x80000
    a.batch, a.q_per_seq, a.num_q_heads, a.q_dtype, a.window_left, a.sm_scale = batch, n, hq, q, -1, D ** -0.5
    a.q_token_stride = a.out_token_stride = hq * D
    a.block_table_stride = a.max_blocks_per_seq = 100
    a.max_seq_len, a.total_kv_len = hints
    out = (ctypes.c_int64 * 8)(*([-7] * 8))
    assert lib.xllm_hip_tree_attention_describe(ctypes.byref(d), ctypes.byref(a), out, 7) == status
    if status != _lib.OK:
        return None
    assert out[6] == 0 and out[7] == -7  # zeros behind the last, nothing past the count
    return dict(zip(FORMS, out))


def test_rows_of_a_workgroup(lib):
    for kv in (_lib.BF16, _lib.INT8, _lib.FP8_E4M3):
        for n, hq, rows, groups in ((1, 8, 32, 1), (8, 8, 32, 1), (16, 8, 64, 1), (17, 8, 128, 1), (64, 16, 128, 4)):
            f = describe(lib, 4, n, hq, 2, 128, 16, kv=kv)
            assert (f["rows_per_workgroup"], f["row_groups"]) == (rows, groups), (kv, n, hq)
    assert describe(lib, 4, 17, 8, 2, 256, 16)["rows_per_workgroup"] == 64
    assert describe(lib, 0, 17, 8, 2, 256, 16) == dict.fromkeys(FORMS, 0)


@pytest.mark.parametrize("change", [dict(D=80), dict(bs=8), dict(bs=24), dict(q=_lib.FP32), dict(kv=_lib.FP16), dict(k_cache=0x10008),
                                    dict(stride_slot=2 ** 27), dict(stride_block=2 ** 31)])
def test_what_the_matrix_kernels_do_not_serve(lib, change):
    sizes = dict(D=128, bs=16)
    f = describe(lib, 4, 8, 8, 2, **{**sizes, **change})
    assert f["rows_per_workgroup"] == 0 and f["line_pieces"] == 0


@pytest.mark.parametrize("bs", [16, 64])
def test_scales_far_apart(lib, bs):
    """The matrix kernels hold a token's scale as a 32-bit byte offset within its group of 16 tokens: 15 strides of
    2^32 / 60 floats are the first that do not fit.  (From 2^30 / block_size floats on the generic kernel serves the call.)"""
    for kv in (_lib.INT8, _lib.FP8_E4M3):
        for stride in (71582789, 2 ** 31 // bs - 1, 2 ** 30 // bs):
            assert describe(lib, 4, 8, 8, 2, 128, bs, kv=kv, scale_stride_slot=stride)["rows_per_workgroup"] == 0, stride
        assert describe(lib, 4, 8, 8, 2, 128, bs, kv=kv, scale_stride_slot=2 ** 30 // bs - 1)["rows_per_workgroup"] == 32
    # (strides of a 16-bit cache's scales, if any are given, are nobody's)
    assert describe(lib, 4, 8, 8, 2, 128, bs, scale_stride_slot=2 ** 40)["rows_per_workgroup"] == 32


def test_without_hints(lib):
    # 16-bit caches: the line from 64 (sequence, kv head, row group)s on; 8-bit ones never
    assert describe(lib, 64, 8, 8, 1, 128, 16)["line_pieces"] == 512
    assert describe(lib, 63, 8, 8, 1, 128, 16)["line_pieces"] == 0
    assert describe(lib, 8, 8, 64, 8, 128, 16)["line_pieces"] == 64
    assert describe(lib, 64, 8, 8, 1, 256, 16)["line_pieces"] == 256
    f = describe(lib, 64, 8, 64, 8, 128, 16, kv=_lib.INT8)
    assert (f["line_pieces"], f["chunk_tokens"], f["chunk_slots"]) == (0, 256, 2)
    assert describe(lib, 1025, 8, 8, 1, 128, 16)["line_pieces"] == 0  # (more sequences than the line holds)


def test_hinted_ragged_batches_lie_on_the_line(lib):
    """The sizes of test_ragged_batches_in_equal_pieces with its hints; and a batch of one sequence with rows, which does
    not: its form is chosen without hints in test_gpu_tree_forms.py."""
    for hq, hkv, D, bs, most in ((8, 2, 128, 16, 8), (16, 2, 128, 32, 8), (16, 2, 128, 16, 30), (32, 2, 128, 16, 30), (14, 2, 64, 32, 4),
                                 (14, 2, 64, 32, 8), (28, 2, 64, 16, 20), (4, 2, 256, 16, 8), (24, 3, 256, 64, 15)):
        f = describe(lib, 9, most, hq, hkv, D, bs, hints=(10 ** 6, 6 * 10 ** 6))
        assert f["line_pieces"] == (256 if D == 256 else 512) // hkv, (hq, hkv, D, bs, most)
    assert describe(lib, 9, 2, 4, 1, 64, 16, hints=(10 ** 6, 6 * 10 ** 6))["line_pieces"] == 0
    assert describe(lib, 1000, 3, 4, 1, 64, 16, hints=(10 ** 6, 6 * 10 ** 8))["line_pieces"] == 512


def test_refusals(lib):
    out = (ctypes.c_int64 * 6)()
    assert lib.xllm_hip_tree_attention_describe(None, None, out, 6) == _lib.INVALID_ARGUMENT
    describe(lib, 4, 513, 8, 2, 128, 16, status=_lib.UNSUPPORTED)
    describe(lib, 4, 8, 8, 2, 128, 16, status=_lib.INVALID_ARGUMENT, k_cache=None)
    q, cache = torch.zeros(8, 4, 128, dtype=torch.bfloat16), torch.zeros(4, 2, 16, 128, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(_lib.XllmHipError):
        ops.tree_decode_describe(q, cache, cache, table, lens)
    with pytest.raises(_lib.XllmHipError):
        ops.tree_decode_describe(q, cache, cache, table, lens, q_per_seq=4)  # not on the GPU
