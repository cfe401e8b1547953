"""The forms of tree attention, each with its choice asserted, against the 64-bit oracle.  Bounds as in
test_gpu_tree_attention.py."""
import numpy as np
import pytest
import torch

from oracle import paged_kv_oracle as orc
from xllm_wxh_amd import ops

from helpers import TORCH_KV_DTYPE, TORCH_Q_DTYPE
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


def far_below(kv, q, D, at, gap, n, L, layout="HND", seed=40):
    """One key (token `at`) whose score is `gap` nats above the others' for every row, and whose value row is zero: the
    output is made of weights far below the largest.  An 8-bit cache has one V scale for all tokens, so that its zero row
    is no smaller than the others by its scale."""
    c = TreeCase([n], [L], 8, 2, D, 16, q=q, kv=kv, layout=layout, seed=seed)
    g = torch.Generator().manual_seed(seed)
    qt = (1.0 + 0.25 * torch.randn(n, 8, D, generator=g)).to(TORCH_Q_DTYPE[q])
    c.q_ref, c.q = qt.float().numpy(), qt.to(c.q.device)
    nb = c.k_ref.shape[0]
    kf, vf = 0.2 * torch.randn(nb, 2, 16, D, generator=g), torch.randn(nb, 2, 16, D, generator=g).abs() * 2.0 ** 12
    blk, slot = int(c.table[0, at // 16]), at % 16
    kf[blk, :, slot], vf[blk, :, slot] = gap / D ** 0.5, 0.0
    if kv in ("int8", "fp8"):
        qk, sk = orc.quantize_per_token_head(kf.numpy(), kv)
        one = float(vf.abs().max()) / (127.0 if kv == "int8" else 448.0)
        sv = torch.full((nb, 2, 16), one)
        qv = (vf / one).round().to(torch.int8) if kv == "int8" else (vf / one).to(torch.float8_e4m3fn)
        c.k_ref, c.v_ref = orc.dequantize(qk, sk, kv), (qv.float() * one).numpy()
        tensors = [torch.from_numpy(qk.view(np.uint8)).view(TORCH_KV_DTYPE[kv]), qv, torch.from_numpy(sk), sv]
    else:
        tensors = [kf.to(TORCH_KV_DTYPE[kv]), vf.to(TORCH_KV_DTYPE[kv]), None, None]
        c.k_ref, c.v_ref = tensors[0].float().numpy(), tensors[1].float().numpy()
    c.k, c.v, c.ks, c.vs = (None if t is None else (t.swapaxes(1, 2).contiguous() if layout == "NHD" else t).to(c.q.device) for t in tensors)
    return c


def lost_below(c, D):
    """What fp16's smallest number may cost an element of the output.  A weight is within 2^-11 of its value or within
    2^-25.  Over a fp16 cache the largest weight of 32 tokens that are taken together is at least 2^-13, and that of the row's
    largest token at least 2^10; over an 8-bit cache the row's largest is at least 2^4."""
    L, n = int(c.lens[0]), c.counts[0]
    k, v = (r[0].astype(np.float64) for r in (c.rows(c.k_ref), c.rows(c.v_ref)))
    out = np.zeros((n, 8, D))
    if c.kv == "bf16":  # (bf16 weights have a float's range)
        return out
    for j in range(n):
        sees = np.array([t < L - n or (int(c.mask[j, 0]) >> (t - L + n)) & 1 for t in range(L)], bool)
        for h in range(8):
            x = k[:, h // 4] @ c.q_ref[j, h].astype(np.float64) * c.scale
            p = np.where(sees, np.exp(x - x[sees].max()), 0.0)
            p /= p.sum()
            if c.kv == "fp16":
                tops = np.repeat([p[i:i + 32].max() for i in range(0, L, 32)], 32)[:L]
                tops *= np.where(tops == p.max(), 2.0 ** -35, 2.0 ** -12)
            else:
                tops = np.full(L, p.max() * 2.0 ** -29)
            out[j, h] = (tops * sees) @ np.abs(v[:, h // 4])
    return out


@pytest.mark.parametrize("kv,q", [("fp16", "fp16"), ("int8", "bf16"), ("fp8", "fp16"), ("bf16", "bf16")])
@pytest.mark.parametrize("D,n,place", [(128, 4, 5), (128, 12, 1040), (64, 40, -1), (256, 20, 2066)])
@pytest.mark.parametrize("gap", [10.0, 18.0])
def test_weights_far_below_a_dominant_one(gpu, kv, q, D, n, place, gap):
    """18 nats are 26 bits: such weights were 0 in fp16, and the output with them.  `place` -1: the first drafted token, which
    is masked for some rows."""
    print("case far below", kv, q, D, n, place, gap, flush=True)
    L = 2100
    c = far_below(kv, q, D, L - n if place < 0 else place, gap, n, L)
    want = c.oracle()
    two_u = torch.finfo(TORCH_Q_DTYPE[q]).eps
    ref = (want[0], want[1], want[2] + lost_below(c, D) / two_u, want[3], want[4])
    for hints in (dict(), dict(max_seq_len=L, total_kv_len=L), dict(max_seq_len=10 ** 6, total_kv_len=10 ** 6)):
        c.check(*c.run(**hints), ref=ref)


@pytest.mark.parametrize("gap", [10.0, 20.0])
def test_weights_far_below_on_the_line(gpu, gap):
    """The same over a fp16 cache on the line: the reference point of a row moves, and differs at the joins."""
    c = far_below("fp16", "fp16", 128, 700, gap, 9, 2100, layout="NHD")
    indptr = torch.tensor([0, 9] + [9] * 99, dtype=torch.int32, device=gpu)
    table = torch.cat([c.d_table, c.d_table.new_zeros(99, c.d_table.size(1))])[:100].contiguous()
    lens = torch.cat([c.d_lens, c.d_lens.new_full((99,), 40)])
    kw = dict(q_indptr=indptr, table=table, lens=lens)
    f = ops.tree_decode_describe(c.q, c.k, c.v, table, lens, scale=c.scale, q_indptr=indptr, q_per_seq=9, kv_layout="NHD")
    assert f["line_pieces"] > 0
    want = c.oracle()
    ref = (want[0], want[1], want[2] + lost_below(c, 128) / 2.0 ** -10, want[3], want[4])
    c.check(*c.run(**kw), ref=ref)


def test_scores_that_scatter_widely(gpu):
    """Scores that scatter by ten nats: over a fp16 cache the reference points move up and down all the time."""
    for n in (6, 40):
        c = TreeCase([n, n], [3000, 1777], 8, 2, 128, 16, q="fp16", kv="fp16", seed=41, std=10.0)
        want = c.oracle()
        c.check(*c.run(), ref=want)
        c.check(*c.run(max_seq_len=3000, total_kv_len=4777), ref=want)


def poisoned(c, victims):
    """Runs the case clean, then with NaN (and infinities) in the V and K rows of one drafted token per sequence and of
    every slot behind the sequences: rows that do not see the token keep their result, those that do have none."""
    clean, clean_lse = c.run()
    blind = np.ones(c.q.size(0), bool)
    places = []
    for b, n in enumerate(c.counts):
        L = int(c.lens[b])
        end = -(-L // c.bs) * c.bs
        places += [(int(c.table[b, t // c.bs]), t % c.bs) for t in range(L, end)]
        if n > L or victims[b] is None:
            continue
        t, lo = L - n + victims[b], int(c.q_indptr[b])
        places.append((int(c.table[b, t // c.bs]), t % c.bs))
        for j in range(n):
            blind[lo + j] = not (int(c.mask[lo + j, victims[b] // 64]) >> (victims[b] % 64)) & 1
    assert blind.any() and not blind.all()
    blind = torch.from_numpy(blind).to(c.q.device)
    blk, slot = (torch.tensor(x, device=c.q.device) for x in zip(*places))
    u = torch.finfo(c.q.dtype).eps
    for what in (float("nan"),) if c.kv == "fp8" else (float("nan"), float("inf")):
        bad = torch.full((1,), what, device=c.q.device).to(c.k.dtype).view(torch.uint8 if c.kv == "fp8" else torch.int16)
        for cache in (c.v, c.k):
            bits = cache.view(bad.dtype)
            keep = bits.clone()
            bits[blk, :, slot] = bad
            got, lse = c.run()
            assert torch.isfinite(got[blind].float()).all()
            # (the piece is then summed token by token, with the weights' own bits: half a step of the weights and of the
            # output, on either side; V is normal, so sums of its products stay below a few units)
            assert torch.allclose(got[blind].float(), clean[blind].float(), rtol=2 * u, atol=2 * u)
            assert torch.allclose(lse[blind], clean_lse[blind], rtol=1e-5, atol=1e-5)
            if cache is c.v or what != what:
                assert not torch.isfinite(got[~blind].float()).any()
            bits.copy_(keep)


@pytest.mark.parametrize("kv,q", [("bf16", "bf16"), ("fp16", "fp16"), ("fp8", "bf16")])
@pytest.mark.parametrize("n,L,victims,Hq,D", [(6, 259, (1, 4), 8, 128), (12, 262, (3, 8), 8, 128), (40, 275, (5, 35), 8, 128), (20, 266, (2, 15), 4, 256),
                                              (12, 520, (2, 9), 14, 64)])
def test_unseen_places_on_both_sides_of_a_cut(gpu, kv, q, n, L, victims, Hq, D):
    """The drafted range lies across the chunks' border at a multiple of 256 tokens; merged afterwards."""
    print("case poison cut", kv, n, D, flush=True)
    for victim in victims:
        c = TreeCase([n], [L], Hq, 2, D, 16, q=q, kv=kv, seed=60 + n)
        f = form_of(c)
        assert f["line_pieces"] == 0 and f["chunk_tokens"] == 256 and f["chunk_slots"] > 1 and (L - n) // 256 < (L - 1) // 256
        poisoned(c, [victim])


@pytest.mark.parametrize("q", ["bf16", "fp16"])
@pytest.mark.parametrize("Hq,D,most", [(8, 128, 8), (8, 128, 13), (16, 128, 20), (14, 64, 4), (8, 256, 20)])
def test_unseen_places_on_the_line(gpu, q, Hq, D, most):
    print("case poison line", q, Hq, D, most, flush=True)
    counts, lens = ragged(34, most, 300, most + 1)
    lens = np.maximum(lens, counts)
    c = TreeCase(counts, lens, Hq, 2, D, 16, q=q, kv=q, seed=70 + most)
    assert form_of(c)["line_pieces"] > 0
    poisoned(c, [None if n < 2 else n // 2 for n in counts])


@pytest.mark.parametrize("kv", ["int8", "fp8"])
@pytest.mark.parametrize("every", [1, 2])
def test_scales_of_zero(gpu, kv, every):
    """Tokens whose scales are zero (a cache that was never written): their score is 0 and they add nothing, but they keep
    their share of the weights' sum.  `every` 1: all tokens are so, and the output is zero, up to this: a V scale below 2^-100 may
    count as 2^-100, and |V| is at most 448 before its scale, so an element may be off by 448 * 2^-100 = 3.5e-28."""
    little = 448 * 2.0 ** -100
    for n, L in ((6, 6000), (20, 700), (40, 6000)):
        print("case scales of zero", kv, every, n, flush=True)
        c = TreeCase([n], [L], 8, 2, 128, 16, kv=kv, seed=36)
        for t in (c.ks, c.vs):
            t[:, :, ::every] = 0.0
        c.k_ref[:, :, ::every], c.v_ref[:, :, ::every] = 0.0, 0.0
        want = c.oracle()
        ref = (want[0], want[1], want[2] + little / 2.0 ** -7, want[3], want[4])  # (2^-7: twice half a step of bf16)
        for hints in (dict(), dict(max_seq_len=L, total_kv_len=L)):
            out, lse = c.run(**hints)
            c.check(out, lse, ref=ref)
            if every == 1:
                assert float(out.float().abs().max()) <= little
