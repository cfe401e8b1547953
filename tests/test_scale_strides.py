"""Scale tensors of a quantised cache whose slots lie far apart (slot-major ones of a very large cache): the matrix kernels
of the decode path hold a scale's place as 32 bits of bytes, so the host gives them no call in which it needs more."""
import ctypes

import pytest
import torch

from xllm_wxh_amd import _lib, ops

from test_gpu_tree_attention import TreeCase


@pytest.mark.parametrize("head_dim,bs,name", [(128, 16, b"mfma_d128"), (64, 32, b"mfma_d64"), (256, 128, b"mfma_d256")])
@pytest.mark.parametrize("kv", [_lib.INT8, _lib.FP8_E4M3])
def test_decode_variant(head_dim, bs, name, kv):
    lib = _lib.load()
    d, a = _lib.KvCacheDesc(), _lib.DecodeArgs()
    d.k_cache, d.v_cache, d.k_scale, d.v_scale = 0x10000, 0x20000, 0x30000, 0x40000
    d.num_blocks, d.block_size, d.num_kv_heads, d.head_dim, d.dtype = 1000, bs, 2, head_dim, kv
    d.stride_block, d.stride_head, d.stride_slot = 2 * bs * head_dim, bs * head_dim, head_dim
    d.scale_stride_block, d.scale_stride_head = 2, 1
    a.q, a.out, a.block_table, a.seq_lens = 0x50000, 0x60000, 0x70000, 0x80000
    a.batch, a.q_per_seq, a.num_q_heads, a.q_dtype, a.window_left, a.sm_scale = 4, 1, 8, _lib.BF16, -1, 0.1
    a.q_token_stride = a.out_token_stride = 8 * head_dim
    a.block_table_stride = a.max_blocks_per_seq = 100
    for stride, want in ((1, name), (2 ** 30 // bs - 1, name), (2 ** 30 // bs, b"generic"), (2 ** 31 // bs - 1, b"generic")):
        d.scale_stride_slot = stride
        assert lib.xllm_hip_paged_decode_variant(ctypes.byref(d), ctypes.byref(a)) == want, stride


@pytest.mark.gpu
@pytest.mark.parametrize("stride", [71582789, 2 ** 26 - 1])
@pytest.mark.parametrize("kv", ["int8", "fp8"])
def test_decode_with_far_scales(gpu, kv, stride):
    print("case decode far scales", kv, stride, flush=True)
    c = TreeCase([1, 1], [90, 41], 8, 2, 128, 16, kv=kv, seed=35)  # (one row per sequence: plain decode)
    far = []
    for t in (c.ks, c.vs):
        store = torch.empty(15 * stride + t.size(0) * 2, dtype=torch.float32, device=gpu)
        view = store.as_strided((t.size(0), 2, 16), (2, 1, stride))
        view.copy_(t)
        far.append(view)
    out = torch.zeros_like(c.q)
    lse = torch.zeros(c.q.size(0), c.Hq, device=gpu)
    ops.batch_decode(c.q, c.k, out, c.d_table, c.d_lens, c.v, output_lse=lse, scale=c.scale, k_cache_quant_scale=far[0],
                     v_cache_quant_scale=far[1])
    c.check(out, lse)
