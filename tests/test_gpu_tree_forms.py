"""The forms of tree attention, each with its choice asserted, against the 64-bit oracle.  Bounds as in
test_gpu_tree_attention.py."""
import numpy as np
import pytest
import torch

from xllm_wxh_amd import ops

from test_gpu_tree_attention import TreeCase

pytestmark = pytest.mark.gpu


def form_of(c, **kw):
    return ops.tree_decode_describe(c.q, c.k, c.v, c.d_table, c.d_lens, scale=c.scale, q_indptr=c.d_indptr, q_per_seq=max(c.counts),
                                    k_cache_quant_scale=c.ks, v_cache_quant_scale=c.vs, kv_layout=c.layout, **kw)


def ragged(batch, most, top, seed):
    """Counts up to `most`, lengths up to `top`: some sequences without rows, some without tokens, some with more rows than
    tokens, one that spans many pieces."""
    rng = np.random.default_rng(seed)
    counts, lens = rng.integers(0, most + 1, batch), rng.integers(0, top, batch)
    counts[[0, batch // 2]], lens[[0, batch // 2]] = most, (top, 2 * top + 3)
    counts[5], lens[6], lens[7] = 0, 0, 1
    return counts.tolist(), lens


@pytest.mark.parametrize("q,layout", [("bf16", "NHD"), ("fp16", "HND")])
@pytest.mark.parametrize("Hq,Hkv,D,bs,most,rows", [(8, 2, 128, 16, 8, 32), (8, 2, 128, 32, 13, 64), (16, 2, 128, 16, 20, 128),
                                                   (14, 2, 64, 32, 4, 32), (14, 2, 64, 16, 20, 128), (8, 2, 256, 16, 20, 64)])
def test_line_without_hints(gpu, q, layout, Hq, Hkv, D, bs, most, rows):
    print("case line without hints", q, Hq, D, most, flush=True)
    counts, lens = ragged(34, most, 300, most)
    c = TreeCase(counts, lens, Hq, Hkv, D, bs, q=q, kv=q, layout=layout, seed=31)
    f = form_of(c)
    assert f["line_pieces"] > 0 and f["rows_per_workgroup"] == rows, f
    c.check(*c.run())


def test_line_of_one_sequence_with_rows(gpu):
    """All but the last sequence are skipped: they have lengths, but no rows."""
    c = TreeCase([0] * 70 + [2], [5] * 70 + [777], 4, 1, 64, 16, seed=32)
    assert form_of(c)["line_pieces"] > 0
    c.check(*c.run())


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("n,Hkv,rows", [(8, 2, 32), (16, 2, 64), (40, 2, 128)])
def test_chunks_without_hints(gpu, kv, n, Hkv, rows):
    print("case chunks without hints", kv, n, flush=True)
    c = TreeCase([n, n - 1], [1300, 2049], 4 * Hkv, Hkv, 128, 16, kv=kv, seed=33)
    f = form_of(c)
    assert f["line_pieces"] == 0 and f["rows_per_workgroup"] == rows and f["chunk_tokens"] == 256 and f["chunk_slots"] > 5, f
    c.check(*c.run())


@pytest.mark.parametrize("stride,rows", [(71582789, 0), (2 ** 26 - 1, 32)])
@pytest.mark.parametrize("kv", ["int8", "fp8"])
def test_scales_far_apart(gpu, kv, stride, rows):
    """Slot-major scale tensors of a very large cache: the scales of a block's 16 tokens lie up to 4.3 GB apart, past 32
    bits of bytes, or just within."""
    print("case far scales", kv, stride, flush=True)
    c = TreeCase([6, 3], [90, 41], 8, 2, 128, 16, kv=kv, seed=34)
    nb = c.ks.size(0)
    far = []
    for t in (c.ks, c.vs):
        store = torch.empty(15 * stride + nb * 2, dtype=torch.float32, device=gpu)
        view = store.as_strided((nb, 2, 16), (2, 1, stride))
        view.copy_(t)
        far.append(view)
    c.ks, c.vs = far
    assert form_of(c)["rows_per_workgroup"] == rows
    c.check(*c.run())
