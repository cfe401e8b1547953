"""What the operators of a tree step refuse, through the C ABI with made-up pointers (nothing is launched) and through
the Python mirror with CPU tensors; the oracle against small known answers."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import tree_step_oracle as tro
from xllm_wxh_amd import _lib, ops
from xllm_wxh_amd import build as xbuild


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        xbuild.build_library(verbose=False)
    return _lib.load()


def refused(lib, status, text, rc):
    assert rc == status, (rc, lib.xllm_hip_last_error())
    assert text.encode() in lib.xllm_hip_last_error(), lib.xllm_hip_last_error()


def step_args():
    a = _lib.StepArgs()
    for i, name in enumerate(("cached_lens", "block_pool", "block_table", "seq_lens", "q_indptr", "slot_mapping", "positions")):
        setattr(a, name, 0x100000 * (i + 1))
    a.pool_rows, a.pool_width, a.pool_stride, a.batch, a.block_size = 4, 8, 8, 4, 16
    a.table_width, a.table_stride, a.num_rows = 8, 8, 4
    return a


STEP = [
    (dict(batch=5000), _lib.UNSUPPORTED, "larger than 4096"),
    (dict(batch=-1), _lib.INVALID_ARGUMENT, "negative"),
    (dict(block_size=0), _lib.INVALID_ARGUMENT, "must be positive"),
    (dict(pool_stride=7), _lib.INVALID_ARGUMENT, "smaller than the row"),
    (dict(table_stride=3), _lib.INVALID_ARGUMENT, "smaller than the row"),
    (dict(q_per_seq=-1), _lib.INVALID_ARGUMENT, "q_per_seq"),
    (dict(q_indptr=None), _lib.INVALID_ARGUMENT, "q_indptr is NULL"),
    (dict(slot_mapping=None), _lib.INVALID_ARGUMENT, "slot_mapping"),
    (dict(seq_lens=None), _lib.INVALID_ARGUMENT, "seq_lens"),
    (dict(kv_indptr=0x900000), _lib.INVALID_ARGUMENT, "go together"),
    (dict(free_blocks=0x900000), _lib.INVALID_ARGUMENT, "free_blocks and free_head"),
    (dict(free_blocks=0x900000, free_head=0xa00000), _lib.INVALID_ARGUMENT, "needs held_blocks"),
    (dict(held_blocks=0x900000), _lib.INVALID_ARGUMENT, "go together"),
    (dict(seq_lens=0x100000), _lib.INVALID_ARGUMENT, "overlaps an input"),
    (dict(slot_mapping=0x200000 + 4 * 31), _lib.INVALID_ARGUMENT, "overlaps an input"),
    (dict(held_blocks=0x900000, held_blocks_out=0x900004, free_head_out=0xb00000), _lib.INVALID_ARGUMENT, "overlaps an input"),
]


@pytest.mark.parametrize("case", range(len(STEP)))
def test_step_indices_refusals(lib, case):
    change, status, text = STEP[case]
    a = step_args()
    for k, v in change.items():
        setattr(a, k, v)
    refused(lib, status, text, lib.xllm_hip_build_step_indices(ctypes.byref(a), None))
    refused(lib, _lib.INVALID_ARGUMENT, "NULL", lib.xllm_hip_build_step_indices(None, None))


def test_tree_masks_refusals(lib):
    call = lambda *a: lib.xllm_hip_tree_masks(*a)  # noqa: E731
    P = 0x1000
    refused(lib, _lib.INVALID_ARGUMENT, "negative", call(P, P, None, -1, 0, 4, P, 1, 1, None, 0, 1, 0, None))
    refused(lib, _lib.INVALID_ARGUMENT, "at least one word", call(P, P, None, 1, 0, 4, P, 1, 0, None, 0, 1, 0, None))
    refused(lib, _lib.INVALID_ARGUMENT, "at least one word", call(P, P, None, 1, 0, 4, P, 1, 2, None, 0, 1, 0, None))
    refused(lib, _lib.UNSUPPORTED, "larger than 8", call(P, P, None, 1, 0, 4, P, 9, 9, None, 0, 1, 0, None))
    refused(lib, _lib.INVALID_ARGUMENT, "NULL", call(None, P, None, 1, 0, 4, P, 1, 1, None, 0, 1, 0, None))
    refused(lib, _lib.INVALID_ARGUMENT, "exceeds", call(P, None, None, 2, 3, 4, P, 1, 1, None, 0, 1, 0, None))
    refused(lib, _lib.INVALID_ARGUMENT, "axes", call(P, P, None, 1, 0, 4, P, 1, 1, P, 0, 5, 4, None))
    refused(lib, _lib.INVALID_ARGUMENT, "axes", call(P, P, None, 1, 0, 4, P, 1, 1, P, 0, 2, 3, None))
    assert call(None, None, None, 0, 0, 4, None, 1, 1, None, 0, 1, 0, None) == _lib.OK


def kv_desc(dtype=_lib.BF16, head_dim=128):
    d = _lib.KvCacheDesc()
    d.k_cache, d.v_cache = 0x10000, 0x20000
    d.num_blocks, d.block_size, d.num_kv_heads, d.head_dim, d.dtype = 4, 16, 2, head_dim, dtype
    d.stride_block, d.stride_head, d.stride_slot = 2 * 16 * head_dim, 16 * head_dim, head_dim
    return d


def tree_args():
    a = _lib.DecodeArgs()
    a.q, a.out, a.block_table, a.seq_lens = 0x30000, 0x40000, 0x50000, 0x60000
    a.batch, a.q_per_seq, a.num_q_heads, a.q_dtype, a.window_left, a.sm_scale = 2, 3, 4, _lib.BF16, -1, 1.0
    a.q_token_stride = a.out_token_stride = 4 * 128
    a.block_table_stride = a.max_blocks_per_seq = 4
    return a


TREE = [
    (dict(), dict(window_left=4), _lib.UNSUPPORTED, "sliding window"),
    (dict(), dict(host_plan=1), _lib.UNSUPPORTED, "host_plan"),
    (dict(head_dim=512), dict(), _lib.UNSUPPORTED, "larger than 256"),
    (dict(), dict(q_per_seq=513), _lib.UNSUPPORTED, "larger than 512"),
    (dict(), dict(num_q_heads=3), _lib.INVALID_ARGUMENT, "not a multiple"),
    (dict(), dict(q_dtype=_lib.INT8), _lib.INVALID_ARGUMENT, "query dtype"),
    (dict(dtype=_lib.INT8), dict(), _lib.INVALID_ARGUMENT, "needs k_scale"),
    (dict(dtype=9), dict(), _lib.INVALID_ARGUMENT, "unknown cache dtype"),
    (dict(stride_slot=-128), dict(), _lib.INVALID_ARGUMENT, "negative"),
    (dict(), dict(seq_lens=None), _lib.INVALID_ARGUMENT, "needs seq_lens"),
    (dict(), dict(block_table=None), _lib.INVALID_ARGUMENT, "neither block_table"),
    (dict(), dict(block_table_stride=3), _lib.INVALID_ARGUMENT, "block_table shape"),
    (dict(), dict(q_token_stride=511), _lib.INVALID_ARGUMENT, "token stride"),
    (dict(), dict(max_seq_len=-1), _lib.INVALID_ARGUMENT, "negative"),
    (dict(), dict(q=None), _lib.INVALID_ARGUMENT, "q, out or tree_mask"),
]


@pytest.mark.parametrize("case", range(len(TREE)))
def test_tree_attention_refusals(lib, case):
    cache, args, status, text = TREE[case]
    d, a = kv_desc(), tree_args()
    for obj, change in ((d, cache), (a, args)):
        for k, v in change.items():
            setattr(obj, k, v)
    refused(lib, status, text, lib.xllm_hip_tree_attention(ctypes.byref(d), ctypes.byref(a), 0x70000, 1, 1, 0x80000, 1 << 30, None))


def test_tree_attention_mask_and_workspace_refusals(lib):
    d, a = kv_desc(), tree_args()
    call = lambda m, s, w, ws, n: lib.xllm_hip_tree_attention(ctypes.byref(d), ctypes.byref(a), m, s, w, ws, n, None)  # noqa: E731
    refused(lib, _lib.INVALID_ARGUMENT, "at least one word", call(0x70000, 0, 1, 0x80000, 1 << 30))
    refused(lib, _lib.UNSUPPORTED, "mask_words", call(0x70000, 9, 9, 0x80000, 1 << 30))
    refused(lib, _lib.INVALID_ARGUMENT, "tree_mask is NULL", call(None, 1, 1, 0x80000, 1 << 30))
    need = lib.xllm_hip_tree_attention_workspace_bytes(2, 3, 4, 2, 128)
    assert need > 0
    refused(lib, _lib.WORKSPACE_TOO_SMALL, "need %d" % need, call(0x70000, 1, 1, 0x80000, need - 1))
    refused(lib, _lib.WORKSPACE_TOO_SMALL, "need", call(0x70000, 1, 1, None, 0))
    refused(lib, _lib.INVALID_ARGUMENT, "256-byte", call(0x70000, 1, 1, 0x80010, 1 << 30))
    a.batch = 0
    assert call(None, 1, 1, None, 0) == _lib.OK


def test_tree_workspace_bounds(lib):
    for sizes in ((1, 1, 1, 1, 1), (1, 512, 64, 8, 128), (4096, 8, 32, 8, 128), (1, 8, 14, 2, 64), (64, 61, 64, 8, 256), (2, 512, 128, 1, 256)):
        assert 0 <= ops.tree_workspace_bytes(*sizes) <= (512 << 20) + 4096, sizes
    assert lib.xllm_hip_tree_attention_workspace_bytes(0, 1, 1, 1, 64) == 0


def test_move_refusals(lib):
    d = kv_desc()
    P = 0x1000

    def call(cache=d, table=P, stride=4, blocks=4, cached=0x2000, acc=0x3000, acc_stride=5, width=5, num=0x4000, batch=2, new=None):
        return lib.xllm_hip_move_accepted_tokens(ctypes.byref(cache) if cache is not None else None, table, stride, blocks, cached, acc,
                                                 acc_stride, width, num, batch, new, None)
    refused(lib, _lib.INVALID_ARGUMENT, "cache is NULL", call(cache=None))
    refused(lib, _lib.INVALID_ARGUMENT, "negative", call(batch=-1))
    refused(lib, _lib.UNSUPPORTED, "larger than 1024", call(width=1025, acc_stride=1025))
    refused(lib, _lib.INVALID_ARGUMENT, "NULL", call(num=None))
    refused(lib, _lib.INVALID_ARGUMENT, "block_table shape", call(stride=3))
    refused(lib, _lib.INVALID_ARGUMENT, "accepted shape", call(acc_stride=4))
    refused(lib, _lib.INVALID_ARGUMENT, "overlaps cached_lens", call(new=0x2004))
    refused(lib, _lib.INVALID_ARGUMENT, "overlaps num_accepted", call(new=0x4000))
    refused(lib, _lib.INVALID_ARGUMENT, "overlaps accepted", call(new=0x3000 + 4 * 9))
    refused(lib, _lib.INVALID_ARGUMENT, "overlaps block_table", call(new=0x1000 + 4 * 7))
    refused(lib, _lib.INVALID_ARGUMENT, "needs k_scale", call(cache=kv_desc(_lib.INT8)))
    assert call(batch=0) == _lib.OK


def test_mrope_refusals(lib):
    a, m = _lib.RopeArgs(), _lib.Mrope()
    a.qkv, a.cos_sin_cache, a.positions = 0x1000, 0x2000, 0x3000
    a.token_stride, a.num_tokens, a.num_q_heads, a.num_k_heads, a.num_v_heads = 512, 3, 2, 1, 1
    a.head_dim = a.rotary_dim = 128
    a.max_position = 10
    m.num_axes, m.axis_stride = 3, 3
    m.sections[0], m.sections[1], m.sections[2] = 24, 20, 20
    call = lambda cache=None, slots=None: lib.xllm_hip_mrope_kv_write(ctypes.byref(a), ctypes.byref(m), cache, slots, None)  # noqa: E731
    m.sections[2] = 19
    refused(lib, _lib.INVALID_ARGUMENT, "63 pairs", call())
    m.sections[2], m.sections[1] = 64, -24
    refused(lib, _lib.INVALID_ARGUMENT, "section 1 is negative", call())
    m.sections[1], m.sections[2], m.num_axes = 20, 20, 5
    refused(lib, _lib.INVALID_ARGUMENT, "num_axes", call())
    m.num_axes, m.axis_stride = 3, 2
    refused(lib, _lib.INVALID_ARGUMENT, "axis_stride", call())
    m.axis_stride = 3
    d = kv_desc()
    refused(lib, _lib.INVALID_ARGUMENT, "slot_mapping is NULL", call(ctypes.byref(d), None))
    refused(lib, _lib.INVALID_ARGUMENT, "cache is [2 heads", call(ctypes.byref(d), 0x4000))
    a.token_stride = 511
    refused(lib, _lib.INVALID_ARGUMENT, "token stride", call())
    a.num_tokens = 0
    assert call() == _lib.OK


def test_python_mirror_refuses():
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)  # noqa: E731
    l = lambda *n: torch.zeros(*n, dtype=torch.int64)  # noqa: E731
    good = dict(cached_lens=i(2), block_pool=i(2, 4), block_size=16, block_table=i(2, 4), seq_lens=i(2), q_indptr=i(3), slot_mapping=i(2),
                positions=l(2))
    for change in (dict(seq_lens=i(3)), dict(q_indptr=i(2)), dict(cached_lens=l(2)), dict(block_table=i(3, 4)), dict(positions=l(3)),
                   dict(slot_mapping=i(4)[::2]), dict(new_lens=i(1)), dict(held_blocks=i(2)), dict(free_blocks=i(4)),
                   dict(paged_kv_indptr=i(3)), dict(block_pool=i(1, 4)), dict(positions=torch.zeros(2)), dict()):
        with pytest.raises(_lib.XllmHipError):
            ops.build_step_indices(**{**good, **change})
    for args, kw in (((i(4), l(4, 1)), dict()), ((i(4), l(4, 1)), dict(q_indptr=i(2), q_per_seq=2)), ((i(4), l(3, 1)), dict(q_per_seq=2)),
                     ((i(4), i(4, 1)), dict(q_per_seq=2)), ((i(4), l(4, 1)), dict(q_per_seq=3)), ((i(4), l(4, 1), l(3)), dict(q_per_seq=2)),
                     ((i(4), l(4, 1), l(4), i(3)), dict(q_per_seq=2)), ((i(4), l(4, 1), l(4), i(2)), dict(q_per_seq=2))):
        with pytest.raises(_lib.XllmHipError):
            ops.tree_masks(*args, **kw)
    bf = lambda *n: torch.zeros(*n, dtype=torch.bfloat16)  # noqa: E731
    cache = bf(4, 2, 16, 128)
    good = dict(query=bf(4, 4, 128), k_cache=cache, v_cache=cache.clone(), output=bf(4, 4, 128), block_table=i(2, 3), seq_lens=i(2),
                tree_mask=l(4, 1), scale=1.0, q_per_seq=2)
    for change in (dict(q_per_seq=None), dict(tree_mask=l(3, 1)), dict(tree_mask=i(4, 1)), dict(block_table=None), dict(v_cache=None),
                   dict(k_cache_quant_scale=torch.zeros(4, 2, 16)), dict(query=bf(4, 512)), dict()):
        with pytest.raises(_lib.XllmHipError):
            ops.batch_tree_decode(**{**good, **change})
    with pytest.raises(_lib.XllmHipError):
        ops.move_accepted_tokens(cache, cache.clone(), i(2, 3), i(2), i(3, 4), i(2))
    with pytest.raises(_lib.XllmHipError):
        ops.move_accepted_tokens(cache, cache.clone(), i(2, 3), i(2), i(2, 4), i(2))  # not on the GPU
    for change in (dict(position_ids=l(3, 5)), dict(mrope_section=[32, 32]), dict(v_cache=None), dict(q_weight=bf(128)), dict(slot_mapping=i(3)),
                   dict(position_ids=torch.zeros(3, 4)), dict(num_heads_q=9), dict()):
        with pytest.raises(_lib.XllmHipError):
            ops.mrope_kv_write(**{**dict(qkv=bf(4, 1024), num_heads_q=4, num_heads_kv=2, head_dim=128, cos_sin_cache=torch.zeros(9, 128),
                                         position_ids=l(3, 4), mrope_section=[24, 20, 20], k_cache=cache, v_cache=cache.clone(),
                                         slot_mapping=i(4)), **change})


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import shutil
    import subprocess
    from test_c_abi_exports import HEADER, _header_struct_fields

    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no gcc")
    structs = {"xllm_hip_step_args": _lib.StepArgs, "xllm_hip_mrope": _lib.Mrope}
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "xllm_hip_paged_kv.h"', "int main(void) {"]
    names = {}
    for cname, cls in structs.items():
        names[cname] = [f.split("[")[0] for f in _fields(HEADER, cname)]
        lines.append('  printf("%%zu\\n", sizeof(%s));' % cname)
        lines += ['  printf("%%zu\\n", offsetof(%s, %s));' % (cname, f) for f in names[cname]]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run([gcc, "-std=c99", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)], check=True)
    out = iter(int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    for cname, cls in structs.items():
        assert next(out) == ctypes.sizeof(cls)
        assert names[cname] == [f[0] for f in cls._fields_]
        for f in names[cname]:
            assert next(out) == getattr(cls, f).offset, (cname, f)


def _fields(header, name):
    import re
    text = re.sub(r"/\*.*?\*/", "", open(header).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    return [re.search(r"([A-Za-z0-9_]+(\[\d+\])?)\s*$", d.strip()).group(1) for d in body.split(";") if d.strip()]


def test_oracle_known_answers():
    # a tree by hand: 0 -> {1, 2}, 2 -> 3; a second sequence of one node
    mask, pos = tro.tree_masks([-1, 0, 0, 2, -1], [0, 4, 5], [10, 7], 1)
    assert mask[:, 0].tolist() == [1, 3, 5, 13, 1] and pos.tolist() == [10, 11, 11, 12, 7]
    pool = np.array([[5, 6, 0], [9, 0, 0]])
    got = tro.step_indices([5, 3], [4, 2], [0, 1], [2, 1], pool, [20, 21, 22], 1, 4, 3, 7)
    assert got["block_table"].tolist() == [[5, 6, 21], [9, 22, 0]] and pool.tolist() == [[5, 6, 21], [9, 22, 0]]
    assert got["slot_mapping"].tolist() == [25, 26, 27, 84, 39, 88, -1] and got["positions"].tolist() == [5, 6, 7, 8, 3, 4, 0]
    assert got["free_head_out"].tolist() == [3, 0] and got["paged_kv_last_page_len"].tolist() == [1, 1]
    assert tro.axis_of_pairs([3, 1, 2], True) == [0, 1, 2, 0, 0, 2] and tro.axis_of_pairs([3, 1, 2], False) == [0, 0, 0, 1, 2, 2]
    # two equal keys seen: the mean of their values; the third is hidden
    q, k = np.ones((1, 1, 2)), [np.ones((3, 1, 2))]
    v = [np.array([[[2.0, 0.0]], [[4.0, 2.0]], [[np.nan, np.nan]]])]
    out, lse, _, _, _ = tro.tree_attention(q, k, v, [0, 1], [3], np.array([[0]], np.uint64), 0.5)
    assert np.allclose(out[0, 0], [3.0, 1.0]) and np.isclose(lse[0, 0], 1.0 / np.log(2.0) + 1.0)
