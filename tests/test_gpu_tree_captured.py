"""A whole tree step captured into one graph — index arrays, masks and positions, rotation and KV write, attention, the
move of the accepted rows — and replayed while the lengths, trees and accepted paths change, with rows behind the last
sequence.  Every replay against the same calls made eagerly on a copy of the state."""
import numpy as np
import pytest
import torch

from xllm_wxh_amd import ops

pytestmark = pytest.mark.gpu

B, HQ, HKV, D, BS, MOST, WIDTH, AXES = 4, 8, 2, 128, 16, 11, 12, 3
ROWS = B * MOST + 5
SECTIONS = [24, 20, 20]


def state(kv, device):
    g = torch.Generator().manual_seed(3)
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32, device=device)  # noqa: E731
    quant = kv == torch.int8
    s = dict(cached=i32(B), new=i32(B), pool=i32(B, WIDTH), held=i32(B), free=torch.randperm(60, generator=g).to(torch.int32).to(device),
             head=i32(1), table=i32(B, WIDTH), lens=i32(B), q_indptr=i32(B + 1), slots=i32(ROWS),
             positions=torch.zeros(ROWS, dtype=torch.int64, device=device), held_out=i32(B), head_out=i32(2), parents=i32(ROWS),
             mask=torch.zeros(ROWS, 1, dtype=torch.int64, device=device),
             # (one tensor per rank: the slots' positions, and those of the axes, zero in the rows behind the last sequence)
             positions_axes=torch.zeros(AXES, ROWS, dtype=torch.int64, device=device),
             qkv=torch.zeros(ROWS, (HQ + 2 * HKV) * D, dtype=torch.bfloat16, device=device),
             out=torch.zeros(ROWS, HQ, D, dtype=torch.bfloat16, device=device), lse=torch.zeros(ROWS, HQ, device=device),
             accepted=i32(B, MOST), count=i32(B), new_lens=i32(B))
    theta = torch.rand(300, D // 2, generator=g) * 6.283
    s["cos_sin"] = torch.cat([theta.cos(), theta.sin()], 1).to(device)
    for name in ("k", "v"):
        s[name] = torch.zeros(60, HKV, BS, D, dtype=kv, device=device)
        s[name + "_scale"] = torch.zeros(60, HKV, BS, device=device) if quant else None
    return s


def step(s):
    ops.build_step_indices(s["cached"], s["pool"], BS, s["table"], s["lens"], s["q_indptr"], s["slots"], s["positions"], new_lens=s["new"],
                           held_blocks=s["held"], free_blocks=s["free"], free_head=s["head"], held_blocks_out=s["held_out"],
                           free_head_out=s["head_out"])
    s["held"].copy_(s["held_out"])
    s["head"].copy_(s["head_out"][:1])
    ops.tree_masks(s["parents"], s["mask"], s["positions_axes"], base=s["cached"], q_indptr=s["q_indptr"])
    ops.mrope_kv_write(s["qkv"], HQ, HKV, D, s["cos_sin"], s["positions_axes"], SECTIONS, s["k"], s["v"], s["slots"],
                       k_cache_scale=s["k_scale"], v_cache_scale=s["v_scale"])
    q = s["qkv"][:, :HQ * D].view(ROWS, HQ, D)
    ops.batch_tree_decode(q, s["k"], s["v"], s["out"], s["table"], s["lens"], s["mask"], scale=D ** -0.5, q_indptr=s["q_indptr"],
                          q_per_seq=MOST, output_lse=s["lse"], k_cache_quant_scale=s["k_scale"], v_cache_quant_scale=s["v_scale"])
    ops.move_accepted_tokens(s["k"], s["v"], s["table"], s["cached"], s["accepted"], s["count"], s["new_lens"], k_cache_scale=s["k_scale"],
                             v_cache_scale=s["v_scale"])
    s["cached"].copy_(s["new_lens"])


def drafts(rng, s):
    """The host's part of a step: how many tokens are drafted, their trees and rows, and the path that will be accepted."""
    n = rng.integers(1, MOST + 1, B)
    parents, accepted, count = np.full(ROWS, -1), np.zeros((B, MOST)), np.zeros(B)
    at = 0
    for b in range(B):
        tree = [-1 if j == 0 else int(rng.integers(-1, j)) for j in range(n[b])]
        parents[at:at + n[b]] = tree
        at += n[b]
        node, path = int(rng.integers(0, n[b])), []
        while node >= 0:
            path.append(node)
            node = tree[node]
        accepted[b, :len(path)], count[b] = path[::-1], len(path)
    qkv = torch.from_numpy(rng.standard_normal((ROWS, (HQ + 2 * HKV) * D)).astype(np.float32)).to(torch.bfloat16)
    for name, value in (("new", n), ("parents", parents), ("accepted", accepted), ("count", count)):
        s[name].copy_(torch.from_numpy(np.asarray(value, np.int32)))
    s["qkv"].copy_(qkv)
    return int(n.sum())


def bits(t):
    return t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}[t.element_size()])


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.int8])
def test_whole_step_captured(gpu, kv):
    print("case whole step captured", kv, flush=True)
    s, eager = state(kv, gpu), state(kv, gpu)
    step(state(kv, gpu))  # (kernels are loaded before the capture)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(s)
    for it in range(6):
        used = drafts(np.random.default_rng(it), s)
        assert drafts(np.random.default_rng(it), eager) == used
        s["out"].fill_(3.0)
        eager["out"].fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        step(eager)
        torch.cuda.synchronize()
        for name, value in s.items():
            if value is not None:
                assert torch.equal(bits(value), bits(eager[name])), (it, name)
        assert torch.isfinite(s["out"][:used].float()).all() and not torch.all(s["out"][:used] == 3.0)
        assert torch.all(s["out"][used:] == 3.0) and torch.all(s["slots"][used:] == -1)
        assert int(s["head_out"][1]) == 0 and torch.equal(s["cached"], s["new_lens"])
