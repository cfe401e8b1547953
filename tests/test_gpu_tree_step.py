"""The operators around tree attention on the GPU against the 64-bit oracle — step indices, ancestor masks, the
multi-axis rotary embedding with its KV write, the move of accepted rows — and a run of them together."""
import math

import numpy as np
import pytest
import torch

from oracle import tree_step_oracle as tro
from xllm_wxh_amd import ops

pytestmark = pytest.mark.gpu

TDT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8, "fp8": torch.float8_e4m3fn}


def i32(x, dev):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(x, np.int32))).to(dev)


def raw(t):
    return t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}[t.element_size()])


# ---------------------------------------------------------------------------------------
# step indices
# ---------------------------------------------------------------------------------------

def run_indices(dev, cached, new, block_size, pool, *, request_ids=None, held=None, free=None, head=None, width=None, pad=0,
                cap=None, pos_dtype=torch.int64, q_per_seq=None):
    B = len(cached)
    width = width or pool.shape[1]
    counts = new if new is not None else [q_per_seq] * B
    total = max(0, int(np.maximum(counts, 0).sum()) + pad) if B else pad
    kw = {}
    full = lambda n, dt=torch.int32: torch.full(n, -77, dtype=dt, device=dev)  # noqa: E731
    out = dict(block_table=full((B, width)), seq_lens=full((B,)), q_indptr=full((B + 1,)), slot_mapping=full((total,)),
               positions=full((total,), pos_dtype))
    extra = dict(paged_kv_indptr=full((B + 1,)), paged_kv_indices=full((cap if cap is not None else B * width,)),
                 paged_kv_last_page_len=full((B,)))
    if held is not None:
        extra.update(held_blocks_out=full((B,)), free_head_out=full((2,)))
        kw["held_blocks"] = i32(held, dev)
    if free is not None:
        kw.update(free_blocks=i32(free, dev), free_head=i32([head], dev))
    if request_ids is not None:
        kw["request_ids"] = i32(request_ids, dev)
    if new is not None:
        kw["new_lens"] = i32(new, dev)
    else:
        kw["q_per_seq"] = q_per_seq
    d_pool = i32(pool, dev)
    ops.build_step_indices(i32(cached, dev), d_pool, block_size, *out.values(), **kw, **extra)
    torch.cuda.synchronize()
    host_pool = np.array(pool, np.int64)
    want = tro.step_indices(cached, counts, request_ids if request_ids is not None else range(B), held, host_pool, free, head,
                            block_size, width, total, cap)
    got = {k: v.cpu().numpy() for k, v in {**out, **extra}.items()}
    for name, value in got.items():
        w = want[name]
        if name == "paged_kv_indices":  # entries behind the last stay as they were
            assert np.all(value[len(w):] == -77)
            value = value[:len(w)]
        assert np.array_equal(value, w), name
    assert np.array_equal(d_pool.cpu().numpy(), host_pool)
    return got


@pytest.mark.parametrize("block_size", [1, 16, 24, 128])
@pytest.mark.parametrize("B,top", [(1, 1), (7, 40), (300, 9), (512, 3), (513, 3), (1100, 5), (4096, 2)])
def test_step_indices_with_allocation(gpu, B, top, block_size):
    print("case indices", B, top, block_size, flush=True)
    rng = np.random.default_rng(B + block_size)
    cached, new = rng.integers(0, 6 * top, B), rng.integers(0, top + 1, B)
    held = -(-cached // block_size) + rng.integers(0, 2, B)
    need = np.maximum(-(-(cached + new) // block_size), held)
    width = int(need.max()) + 2
    rows = B + 3
    pool = rng.integers(0, 10 ** 6, (rows, width))
    free = rng.permutation(10 ** 5)[: int((need - held).sum()) + 4]
    run_indices(gpu, cached, new, block_size, pool, request_ids=rng.permutation(rows)[:B], held=held, free=free, head=4, pad=5)


def test_step_indices_plain_forms(gpu):
    rng = np.random.default_rng(0)
    pool = rng.integers(1, 500, (6, 9))
    run_indices(gpu, [5, 0, 31, 64, 7, 0], None, 8, pool, q_per_seq=1, pos_dtype=torch.int32)
    run_indices(gpu, [5, 0, 31, 60, 7, 0], [3, 0, 2, 1, 20, 0], 8, pool, request_ids=[2, 2, 2, 0, 1, 5])  # rows may repeat
    run_indices(gpu, [5], [0], 8, pool, pad=3)
    run_indices(gpu, [], None, 8, pool, q_per_seq=4, pad=3)
    run_indices(gpu, [5000, 3, 900], [2100, 1, 1500], 2, rng.integers(1, 500, (3, 4000)), pad=1)  # several tiles of rows and columns


def test_step_indices_when_something_is_missing(gpu):
    rng = np.random.default_rng(1)
    pool = rng.integers(1, 500, (5, 6))
    # the free list ends in the middle of the third sequence; the head may lie past its end
    for free in ([9, 8, 7, 6], [9], []):
        for head in (0, 2, 6):
            run_indices(gpu, [8, 8, 8, 0], [9, 1, 20, 4], 4, pool, request_ids=[4, 0, 2, 1], held=[2, 2, 2, 0], free=free, head=head)
    # no free list; a table and a pool narrower than the lengths; ids and lengths out of range
    run_indices(gpu, [8, 30, 40], [9, 1, 2], 4, pool, held=[2, 6, 6])
    run_indices(gpu, [8, 30, 40], [9, 1, 2], 4, pool, width=3, cap=5)
    run_indices(gpu, [8, -3, 4], [9, 3, -2], 4, pool, request_ids=[-1, 77, 4], held=[-2, 1, 99], free=[11, 12, 13], head=0)
    pool[1, 0], pool[2, 1] = -5, 2 ** 30
    run_indices(gpu, [0, 0, 7], [4, 3, 9], 4, pool)


def test_step_indices_captured(gpu):
    """Replays read the lengths of their time, after the step's own outputs became the next one's inputs."""
    B, bs = 5, 4
    rng = np.random.default_rng(2)
    pool = np.zeros((B, 40), np.int64)
    d_pool = i32(pool, gpu)
    free = rng.permutation(300)
    cached, new, held, head = (torch.zeros(B, dtype=torch.int32, device=gpu) for _ in range(4))
    head = head[:1].clone()
    table, lens, indptr = torch.zeros(B, 40, dtype=torch.int32, device=gpu), torch.zeros_like(cached), torch.zeros(B + 1, dtype=torch.int32, device=gpu)
    slots, pos = torch.zeros(64, dtype=torch.int32, device=gpu), torch.zeros(64, dtype=torch.int64, device=gpu)
    held_out, head_out = torch.zeros_like(held), torch.zeros(2, dtype=torch.int32, device=gpu)
    d_free = i32(free, gpu)

    def step():
        ops.build_step_indices(cached, d_pool, bs, table, lens, indptr, slots, pos, new_lens=new, held_blocks=held, free_blocks=d_free,
                               free_head=head, held_blocks_out=held_out, free_head_out=head_out)
        held.copy_(held_out)
        head.copy_(head_out[:1])
        cached.copy_(lens)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    c, h, at = np.zeros(B, np.int64), np.zeros(B, np.int64), 0
    for it in range(6):
        n = rng.integers(0, 9, B)
        new.copy_(i32(n, gpu))
        g.replay()
        torch.cuda.synchronize()
        want = tro.step_indices(c, n, range(B), h, pool, free, at, bs, 40, 64)
        assert np.array_equal(table.cpu().numpy(), want["block_table"]) and np.array_equal(slots.cpu().numpy(), want["slot_mapping"])
        assert np.array_equal(pos.cpu().numpy(), want["positions"]) and np.array_equal(d_pool.cpu().numpy(), pool)
        c, h, at = want["seq_lens"], want["held_blocks_out"], int(want["free_head_out"][0])


# ---------------------------------------------------------------------------------------
# ancestor masks
# ---------------------------------------------------------------------------------------

def parents_of(kind, n, rng):
    if kind == "chain":
        return [j - 1 for j in range(n)]
    if kind == "backward":  # children in front of their parents
        return [j + 1 if j + 1 < n else -1 for j in range(n)]
    if kind == "star":
        return [-1 if j == 0 else 0 for j in range(n)]
    if kind == "bad":  # cycles, parents that are no nodes
        return [int(x) for x in rng.integers(-3, n + 3, n)]
    return [-1 if j == 0 else int(rng.integers(-1, j)) for j in range(n)]


@pytest.mark.parametrize("kind", ["tree", "chain", "backward", "star", "bad"])
@pytest.mark.parametrize("counts,words", [([1], 1), ([16, 5, 64, 0, 63], 1), ([65, 128, 3], 2), ([200, 130], 4), ([512, 300, 77], 8),
                                          ([70, 10], 1)])
def test_tree_masks(gpu, kind, counts, words):
    print("case masks", kind, counts, flush=True)
    rng = np.random.default_rng(3)
    parents = np.concatenate([parents_of(kind, n, rng) for n in counts if n] + [[-1, 0, 1]])  # three rows of no sequence
    indptr = np.concatenate([[0], np.cumsum(counts)])
    base = rng.integers(0, 9000, len(counts))
    rows = len(parents)
    mask = torch.full((rows, words + 2), 123, dtype=torch.int64, device=gpu)
    pos = torch.full((3, rows), -9, dtype=torch.int64, device=gpu)
    ops.tree_masks(i32(parents, gpu), mask[:, 1:1 + words], pos, i32(base, gpu), q_indptr=i32(indptr, gpu))
    want, want_pos = tro.tree_masks(parents, indptr, base, words)
    n = int(indptr[-1])
    got = mask.cpu().numpy()
    if kind != "bad":
        assert np.all(got[:, 0] == 123) and np.all(got[:, -1] == 123) and np.all(got[n:] == 123)
        assert np.array_equal(got[:n, 1:-1].view(np.uint64), want[:n])
        for a in range(3):
            assert np.array_equal(pos[a].cpu().numpy()[:n], want_pos[:n])
        assert torch.all(pos[:, n:] == -9)
    else:
        # nodes whose chain ends at the context have exact masks; of the others only that bits stay in range is promised
        for b in range(len(counts)):
            lo, hi = indptr[b], indptr[b + 1]
            limit = min(hi - lo, 64 * words)
            for v in range(limit):
                seen, at = set(), v
                while 0 <= at < limit and at not in seen:
                    seen.add(at)
                    at = int(parents[lo + at])
                if not 0 <= at < limit:
                    assert np.array_equal(got[lo + v, 1:-1].view(np.uint64), want[lo + v])
                    assert int(pos[0, lo + v]) == want_pos[lo + v]


def test_tree_masks_uniform_and_int32(gpu):
    rng = np.random.default_rng(4)
    parents = np.concatenate([parents_of("tree", 33, rng) for _ in range(6)])
    indptr = np.arange(7) * 33
    mask, pos = torch.zeros(198, 1, dtype=torch.int64, device=gpu), torch.zeros(198, dtype=torch.int32, device=gpu)
    ops.tree_masks(i32(parents, gpu), mask, pos, q_per_seq=33)
    want, want_pos = tro.tree_masks(parents, indptr, None, 1)
    assert np.array_equal(mask.cpu().numpy().view(np.uint64), want) and np.array_equal(pos.cpu().numpy(), want_pos)
    mask.zero_()
    ops.tree_masks(i32(parents, gpu), mask, q_indptr=i32(indptr, gpu))  # positions are optional
    assert np.array_equal(mask.cpu().numpy().view(np.uint64), want)


# ---------------------------------------------------------------------------------------
# multi-axis rotary embedding + KV write
# ---------------------------------------------------------------------------------------

def rope_inputs(T, hq, hkv, D, R, axes, kind, seed, table_kind="fp32", extra=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, (hq + 2 * hkv) * D + extra, generator=g).to(TDT[kind])
    w = [(torch.rand(D, generator=g) + 0.5).to(TDT[kind]) for _ in range(2)]
    theta = torch.rand(300, R // 2, generator=g) * 6.283
    table = torch.cat([theta.cos(), theta.sin()], 1).to(TDT[table_kind])
    pos = torch.randint(-2, 303, (axes, T), generator=g)  # some outside the table: clamped
    return qkv, w, table, pos


def sections_for(axes, half):
    part = [half // (axes + 1)] * axes
    part[0] += half - sum(part)
    return part


ROPE = [
    # T, hq, hkv, D, R, axes, kind, norm, interleave, table type
    (1, 14, 2, 64, 64, 3, "fp16", False, False, "fp32"),
    (33, 32, 8, 128, 128, 3, "bf16", True, False, "fp32"),
    (700, 32, 8, 128, 128, 3, "bf16", True, False, "bf16"),  # the form for many tokens
    (17, 8, 4, 128, 64, 2, "bf16", True, True, "bf16"),       # partial rotary, neighbouring pairs
    (9, 4, 2, 256, 256, 4, "fp32", True, False, "fp32"),
    (9, 4, 2, 256, 96, 2, "fp16", False, False, "fp16"),      # halves of 48 elements: partners six lanes away
    (5, 3, 1, 80, 80, 3, "bf16", True, False, "fp32"),        # off the vector path
    (5, 3, 1, 128, 24, 2, "fp32", False, True, "fp32"),
    (5, 3, 1, 64, 20, 1, "bf16", True, False, "fp32"),
]


@pytest.mark.parametrize("dealt", [False, True])
@pytest.mark.parametrize("case", range(len(ROPE)))
def test_mrope_matches_oracle(gpu, case, dealt):
    T, hq, hkv, D, R, axes, kind, norm, interleave, table_kind = ROPE[case]
    print("case mrope", case, dealt, flush=True)
    qkv, w, table, pos = rope_inputs(T, hq, hkv, D, R, axes, kind, case, table_kind)
    sec = sections_for(axes, R // 2)
    x = qkv.double().view(T, hq + 2 * hkv, D).numpy()
    args = (pos.numpy(), table.double().numpy(), sec, dealt, interleave)
    want = np.concatenate([tro.mrope(x[:, :hq], *args, w[0].double().numpy() if norm else None),
                           tro.mrope(x[:, hq:hq + hkv], *args, w[1].double().numpy() if norm else None)], 1)
    d = qkv.to(gpu)
    nb, bs = T // 16 + 2, 16
    k, v = (torch.full((nb, hkv, bs, D), 7.0, device=gpu).to(TDT[kind]) for _ in range(2))
    slots = torch.randperm(nb * bs)[:T].to(torch.int32)
    slots[0] = -1 if T > 1 else slots[0]
    ops.mrope_kv_write(d, hq, hkv, D, table.to(gpu), pos.to(gpu), sec, k, v, slots.to(gpu), mrope_interleaved=dealt,
                       q_weight=w[0].to(gpu) if norm else None, k_weight=w[1].to(gpu) if norm else None, interleaved=interleave)
    got = d.double().cpu().numpy().reshape(T, hq + 2 * hkv, D)
    # one rounding to the element type, and float arithmetic on a pair of the head's magnitude: two products, a sum, and
    # with a norm the mean of D squares, a root, a quotient and two products more
    u = torch.finfo(TDT[kind]).eps / 2
    big = np.abs(want).max(-1, keepdims=True) * math.sqrt(2.0)
    tol = u * np.abs(want) + (4 + (D / 2 + 8 if norm else 0)) * 2.0 ** -24 * big + (2.0 ** -25 if kind == "fp16" else 0)
    assert np.all(np.abs(got[:, :hq + hkv] - want) <= tol)
    rows = d.view(T, hq + 2 * hkv, D)
    assert torch.equal(raw(rows[:, hq + hkv:]), raw(qkv.to(gpu).view(T, hq + 2 * hkv, D)[:, hq + hkv:]))
    # the cache holds the new rows where the slots say and is untouched elsewhere
    wk, wv = (torch.full((nb, hkv, bs, D), 7.0, device=gpu).to(TDT[kind]) for _ in range(2))
    for t in range(T):
        s = int(slots[t])
        if s >= 0:
            wk[s // bs, :, s % bs], wv[s // bs, :, s % bs] = rows[t, hq:hq + hkv], rows[t, hq + hkv:]
    assert torch.equal(raw(k), raw(wk)) and torch.equal(raw(v), raw(wv))


@pytest.mark.parametrize("kv", ["int8", "fp8", None])
@pytest.mark.parametrize("D,layout", [(128, "HND"), (64, "NHD"), (80, "HND")])
def test_mrope_with_equal_positions_is_rope(gpu, kv, D, layout):
    """One position on every axis: rope_kv_write's result — the rotated heads, and the quantised rows and scales that
    quant_to_paged_cache makes of them."""
    T, hq, hkv = 40, 6, 2
    qkv, w, table, pos = rope_inputs(T, hq, hkv, D, D, 1, "bf16", 5)
    pos = pos.clamp(0, 299)
    nb, bs = 4, 16
    shape = (nb, hkv, bs, D) if layout == "HND" else (nb, bs, hkv, D)
    slots = torch.randperm(nb * bs)[:T].to(torch.int32).to(gpu)
    res = []
    for axes in (0, 3):
        d = qkv.to(gpu)
        cache = [torch.zeros(shape, dtype=torch.uint8, device=gpu).view(TDT[kv]) for _ in range(2)] if kv else [None, None]
        scale = [torch.zeros(shape[:3], device=gpu) for _ in range(2)] if kv else [None, None]
        kw = dict(q_weight=w[0].to(gpu), k_weight=w[1].to(gpu), k_cache_scale=scale[0], v_cache_scale=scale[1], kv_layout=layout)
        if axes == 0 and kv:
            ops.rope_kv_write(d, hq, hkv, D, table.to(gpu), pos[0].to(gpu), cache[0], cache[1], slots, **kw)
        elif axes == 0:
            ops.fused_qk_norm_rope(d, hq, hkv, hkv, D, 1e-6, w[0].to(gpu), w[1].to(gpu), table.to(gpu), False, pos[0].to(gpu))
        else:
            ops.mrope_kv_write(d, hq, hkv, D, table.to(gpu), pos.to(gpu).expand(3, T).contiguous(), sections_for(3, D // 2), cache[0],
                               cache[1], slots if kv else None, **kw)
            if kv:  # against the quantising write of what stands in qkv
                rows = d.view(T, hq + 2 * hkv, D)
                c2 = [torch.zeros(shape, dtype=torch.uint8, device=gpu).view(TDT[kv]) for _ in range(2)]
                s2 = [torch.zeros(shape[:3], device=gpu) for _ in range(2)]
                ops.quant_to_paged_cache(ops.ReshapePagedCacheParams(key=rows[:, hq:hq + hkv], value=rows[:, hq + hkv:], k_cache=c2[0],
                                                                     v_cache=c2[1], slot_mapping=slots, k_cache_scale=s2[0],
                                                                     v_cache_scale=s2[1], kv_layout=layout))
                for a, b in zip(cache + scale, c2 + s2):
                    assert torch.equal(raw(a), raw(b))
        res.append(d)
    if D == 128:  # (the same order of the squares' sum)
        assert torch.equal(raw(res[0]), raw(res[1]))
    else:
        a, b = res[0].float(), res[1].float()
        assert torch.all((a - b).abs() <= 2.0 ** -7 * a.abs() + 1e-6)


def test_mrope_rounding_each_operation_strides_and_int32(gpu):
    T, hq, hkv, D = 12, 4, 2, 128
    qkv, w, table, pos = rope_inputs(T, hq, hkv, D, D, 1, "bf16", 6, extra=64)
    pos = pos.clamp(0, 299)
    width = (hq + 2 * hkv) * D
    wide = qkv.to(gpu)
    keep = wide[:, width:].clone()
    ops.mrope_kv_write(wide[:, :width], hq, hkv, D, table.to(gpu), pos.to(gpu).expand(2, T).contiguous().to(torch.int32),
                       [32, 32], round_each_op=True)
    want_q = qkv[:, :hq * D].contiguous().to(gpu)
    want_k = qkv[:, hq * D:(hq + hkv) * D].contiguous().to(gpu)
    ops.rotary_embedding(pos[0].to(gpu), want_q, want_k, table.to(gpu), True)
    assert torch.equal(raw(wide[:, :hq * D]), raw(want_q)) and torch.equal(raw(wide[:, hq * D:(hq + hkv) * D]), raw(want_k))
    assert torch.equal(raw(wide[:, width:]), raw(keep))


# ---------------------------------------------------------------------------------------
# accepted rows
# ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("kv,D", [("bf16", 128), ("fp32", 256), ("int8", 128), ("fp8", 64), ("fp16", 72), ("int8", 20), ("bf16", 3)])
@pytest.mark.parametrize("block_size", [16, 12])
def test_move_accepted_tokens(gpu, layout, kv, D, block_size):
    print("case accept", layout, kv, D, block_size, flush=True)
    rng = np.random.default_rng(7)
    B, hkv, width, draft = 9, 3, 11, 40
    cached = rng.integers(0, 50, B)
    cached[0] = 0
    per = -(-(50 + draft) // block_size)
    nb = B * per + 2
    table = (rng.permutation(nb - 2) + 1)[:B * per].reshape(B, per)
    table[8, -1] = nb + 5  # ids outside the cache move nothing
    table[7, 0] = -1
    accepted = rng.integers(0, draft, (B, width))  # any order, repeats among them
    accepted[1] = np.arange(width)                  # nothing to move
    accepted[2] = np.arange(width) + 1              # every destination but the first is a source
    accepted[3] = np.arange(width)[::-1]
    accepted[4, 2], accepted[4, 3] = -1, 10 ** 6    # past the table
    count = rng.integers(0, width + 1, B)
    count[1:5] = width
    count[5], count[6] = -4, width + 9
    shape = (nb, hkv, block_size, D) if layout == "HND" else (nb, block_size, hkv, D)
    eb = torch.empty(0, dtype=TDT[kv]).element_size()
    caches = [torch.randint(0, 255, (*shape[:3], D * eb), dtype=torch.uint8).view(TDT[kv]) for _ in range(2)]
    scales = [torch.rand(shape[:3]) for _ in range(2)] if kv in ("int8", "fp8") else [None, None]
    dev = [t.to(gpu) if t is not None else None for t in caches + scales]
    new = torch.full((B,), -1, dtype=torch.int32, device=gpu)
    ops.move_accepted_tokens(dev[0], dev[1], i32(table, gpu), i32(cached, gpu), i32(accepted, gpu), i32(count, gpu), new,
                             k_cache_scale=dev[2], v_cache_scale=dev[3], kv_layout=layout)
    for host, got in zip(caches + scales, dev):
        if host is None:
            continue
        bits = raw(host).numpy().copy()
        hnd = bits if layout == "HND" else bits.swapaxes(1, 2)

        def at(b, tok):
            blk = int(table[b, tok // block_size])
            return (blk, tok % block_size) if 0 <= blk < nb else None

        def get(b, tok):
            p = at(b, tok)
            return None if p is None else hnd[p[0], :, p[1]].copy()

        def put(b, tok, rows):
            p = at(b, tok)
            hnd[p[0], :, p[1]] = rows
        tro.move_accepted(get, put, cached, accepted, count, width, per * block_size)
        assert np.array_equal(raw(got).cpu().numpy(), bits)
    assert np.array_equal(new.cpu().numpy(), cached + np.clip(count, 0, width))


def test_move_long_paths_and_many_sequences(gpu):
    rng = np.random.default_rng(8)
    for B, width, hkv, D in ((2, 1000, 8, 128), (700, 13, 8, 128), (1, 1, 1, 64)):
        per, bs = -(-(2 * width + 5) // 16), 16
        nb = B * per
        table = rng.permutation(nb).reshape(B, per)
        k, v = (torch.randn(nb, hkv, bs, D, device=gpu).to(torch.bfloat16) for _ in range(2))
        pick = np.sort(np.stack([rng.permutation(2 * width)[:width] for _ in range(B)]), 1)
        cached, count = rng.integers(0, 5, B), rng.integers(0, width + 1, B)
        t = torch.from_numpy(table).to(gpu)
        want = []
        for cache in (k, v):
            w = cache.clone()
            b = np.repeat(np.arange(B), count)
            i = np.concatenate([np.arange(n) for n in count]) if count.sum() else np.zeros(0, np.int64)
            src, dst = cached[b] + pick[b, i], cached[b] + i
            fb, tb = t[b, src // bs], t[b, dst // bs]
            w[tb, :, torch.from_numpy(dst % bs).to(gpu)] = cache[fb, :, torch.from_numpy(src % bs).to(gpu)]
            want.append(w)
        ops.move_accepted_tokens(k, v, i32(table, gpu), i32(cached, gpu), i32(pick, gpu), i32(count, gpu))
        assert torch.equal(k, want[0]) and torch.equal(v, want[1])


# ---------------------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv", ["bf16", "int8"])
def test_speculative_steps_together(gpu, kv):
    """Four steps of three sequences, everything but the drafts on the device: indices from the lengths, masks and
    positions from the parents, rotation and KV write, attention, a path accepted, its rows moved.  After every step
    the rows of the accepted tokens are where a step without drafts would have put them."""
    B, hq, hkv, D, bs, n, bf = 3, 8, 2, 128, 16, 9, torch.bfloat16
    rng = np.random.default_rng(9)
    g = torch.Generator().manual_seed(9)
    nb, width = 60, 16
    quant = kv == "int8"
    k, v = (torch.zeros(nb, hkv, bs, D, dtype=torch.uint8 if quant else bf, device=gpu).view(TDT[kv]) for _ in range(2))
    ks, vs = (torch.zeros(nb, hkv, bs, device=gpu) for _ in range(2)) if quant else (None, None)
    pool, free = torch.zeros(B, width, dtype=torch.int32, device=gpu), i32(rng.permutation(nb), gpu)
    cached, held, head = (torch.zeros(m, dtype=torch.int32, device=gpu) for m in (B, B, 1))
    table, lens, indptr = torch.zeros(B, width, dtype=torch.int32, device=gpu), torch.zeros(B, dtype=torch.int32, device=gpu), torch.zeros(B + 1, dtype=torch.int32, device=gpu)
    slots, pos = torch.zeros(B * n, dtype=torch.int32, device=gpu), torch.zeros(B * n, dtype=torch.int64, device=gpu)
    held_out, head_out = torch.zeros_like(held), torch.zeros(2, dtype=torch.int32, device=gpu)
    mask, pos3 = torch.zeros(B * n, 1, dtype=torch.int64, device=gpu), torch.zeros(3, B * n, dtype=torch.int64, device=gpu)
    theta = torch.rand(256, D // 2, generator=g) * 6.283
    table_cs = torch.cat([theta.cos(), theta.sin()], 1).to(gpu)
    sec = [24, 20, 20]
    history = [[] for _ in range(B)]  # per sequence: (key row, value row) of every token in the cache, dequantised
    offset = i32([0, 3, 7], gpu)      # the sequences' positions run ahead of their lengths
    for step in range(4):
        ops.build_step_indices(cached, pool, bs, table, lens, indptr, slots, pos, q_per_seq=n, held_blocks=held, free_blocks=free,
                               free_head=head, held_blocks_out=held_out, free_head_out=head_out)
        held, head = held_out.clone(), head_out[:1].clone()
        parents = np.concatenate([parents_of("tree", n, rng) for _ in range(B)])
        ops.tree_masks(i32(parents, gpu), mask, pos3, cached + offset, q_per_seq=n)
        qkv = torch.randn(B * n, (hq + 2 * hkv) * D, generator=g).to(bf).to(gpu)
        ops.mrope_kv_write(qkv, hq, hkv, D, table_cs, pos3, sec, k, v, slots, k_cache_scale=ks, v_cache_scale=vs)
        q = qkv[:, :hq * D].view(B * n, hq, D)
        out, lse = torch.zeros(B * n, hq, D, dtype=bf, device=gpu), torch.zeros(B * n, hq, device=gpu)
        ops.batch_tree_decode(q, k, v, out, table, lens, mask, scale=D ** -0.5, q_per_seq=n, output_lse=lse, k_cache_quant_scale=ks,
                              v_cache_quant_scale=vs)
        path = np.zeros((B, n), np.int64)
        count = np.zeros(B, np.int64)
        for b in range(B):  # a path from the context to some node
            at, chain = int(rng.integers(0, n)), []
            while at >= 0:
                chain.append(at)
                at = int(parents[b * n + at])
            path[b, :len(chain)], count[b] = chain[::-1], len(chain)
        # the oracle: what the cache holds is the history, then the drafts as qkv shows them
        rows = qkv.float().view(B, n, hq + 2 * hkv, D).cpu().numpy()
        keys, values = rows[:, :, hq:hq + hkv], rows[:, :, hq + hkv:]
        if quant:
            from oracle import paged_kv_oracle as orc
            deq = lambda x: orc.dequantize(*orc.quantize_per_token_head(x, "int8"), "int8")  # noqa: E731
            keys, values = deq(keys), deq(values)
        k_rows = [np.stack([r[0] for r in history[b]] + list(keys[b])) for b in range(B)]
        v_rows = [np.stack([r[1] for r in history[b]] + list(values[b])) for b in range(B)]
        wmask, wpos = tro.tree_masks(parents, np.arange(B + 1) * n, (cached + offset).cpu().numpy(), 1)
        assert np.array_equal(mask.cpu().numpy().view(np.uint64), wmask) and np.array_equal(pos3[2].cpu().numpy(), wpos)
        want, want_lse, absv, dots, ksum = tro.tree_attention(q.float().cpu().numpy(), k_rows, v_rows, np.arange(B + 1) * n,
                                                              [len(x) for x in k_rows], wmask, D ** -0.5)
        # weights and output rounded to bf16, scores in float (int8: queries may be 16-bit fixed point)
        d = dots * (D + 8) * 2.0 ** -24 + (ksum * float(q.float().abs().max()) * 2.0 ** -16 if quant else 0)
        tol = absv * (2 * d[..., None] + 2 * 2.0 ** -8 + 2.0 ** -13) + 1e-30
        assert np.all(np.abs(out.double().cpu().numpy() - want) <= tol), step
        new = torch.zeros_like(cached)
        ops.move_accepted_tokens(k, v, table, cached, i32(path, gpu), i32(count, gpu), new, k_cache_scale=ks, v_cache_scale=vs)
        for b in range(B):
            history[b] += [(keys[b, i], values[b, i]) for i in path[b, :count[b]]]
        cached = new
        assert cached.tolist() == [len(x) for x in history]
        # the cache read back
        total = sum(len(x) for x in history)
        got_k, got_v = (torch.zeros(total, hkv, D, dtype=bf, device=gpu) for _ in range(2))
        top = max(len(x) for x in history)
        if quant:
            ops.dequant_from_paged_cache(got_k, got_v, k, v, ks, vs, cached, top, None, table)
        else:
            ops.reshape_from_cache(got_k, got_v, k, v, cached, top, None, table)
        at = 0
        for b in range(B):
            m = len(history[b])
            for got, which in ((got_k, 0), (got_v, 1)):
                w = torch.from_numpy(np.stack([r[which] for r in history[b]]).astype(np.float32)).to(bf)
                assert torch.equal(got[at:at + m].cpu(), w), (step, b, which)
            at += m
