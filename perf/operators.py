"""The operators of a speculative step over a tree of drafted tokens on the paged KV cache, as cases that
can be timed and compared: the step's index arrays from request lengths, ancestor masks from parents, the
multi-axis rotary embedding with its KV write, attention under the tree's mask, and the move of the accepted
tokens' cache rows.  Each has a plain form in elementary torch operations (32-bit arithmetic, rounded once) and,
where `own` is true, the framework's call."""
import math

import torch

own = False

DEVICE = "cuda"
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8,
           "fp8": torch.float8_e4m3fn}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1, "fp8": 1}
_GOLDEN = 0.6180339887498949


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------

def listed():
    return [
        # the index arrays of a small decode step: nothing but latency
        dict(name="indices_decode_b8", op="indices", batch=8, new=1, ragged=0.0, cached=4096, block_size=16, pad=0),
        # a mixed step of a busy server: chunks of up to 700 new tokens, 255 sequences, padded for a captured graph
        dict(name="indices_mixed_b255", op="indices", batch=255, new=700, ragged=0.97, cached=9001, block_size=128, pad=61),
        # one small drafted tree per sequence of a small batch
        dict(name="masks_b4_n16", op="masks", batch=4, nodes=16, ragged=0.0),
        # wide dynamic trees, several words to a mask, sequences of different sizes
        dict(name="masks_b192_n300", op="masks", batch=192, nodes=300, ragged=0.8),
        # the drafted tokens of eight sequences, head_dim 64, three axes dealt out in turn
        dict(name="mrope_tree_b8", op="mrope", tokens=8 * 17, q_heads=14, kv_heads=2, head_dim=64, dtype="fp16", norm=False,
             block_size=32, axes=3, dealt=True),
        # a prompt chunk with images, normalised heads, sections side by side
        dict(name="mrope_prompt_8191", op="mrope", tokens=8191, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16", norm=True,
             block_size=16, axes=3, dealt=False),
        # one short sequence verifying a few drafts: latency
        dict(name="attend_b1_n8", op="attend", batch=1, nodes=8, len=311, q_heads=14, kv_heads=2, head_dim=64, q="bf16", kv="bf16",
             block_size=32, ragged=0.0),
        # the ordinary serving step: 64 sequences of 4096 tokens, 8 drafts each
        dict(name="attend_b64_n8", op="attend", batch=64, nodes=8, len=4096, q_heads=32, kv_heads=8, head_dim=128, q="bf16",
             kv="bf16", block_size=16, ragged=0.0),
        # few long sequences over an 8-bit cache: the long axis has to be split
        dict(name="attend_b3_n31_int8", op="attend", batch=3, nodes=31, len=32001, q_heads=32, kv_heads=8, head_dim=128, q="bf16",
             kv="int8", block_size=128, ragged=0.5),
        # large trees under many query heads to a kv head, ragged lengths: as much arithmetic as memory
        dict(name="attend_b24_n61_fp8", op="attend", batch=24, nodes=61, len=8192, q_heads=64, kv_heads=8, head_dim=128, q="bf16",
             kv="fp8", block_size=16, ragged=0.9),
        # the accepted tokens of a small batch
        dict(name="accept_b8", op="accept", batch=8, path=5, nodes=16, cached=700, kv_heads=2, head_dim=64, kv="bf16", block_size=32),
        # a large batch over an 8-bit cache with scales, long paths
        dict(name="accept_b512_fp8", op="accept", batch=512, path=13, nodes=61, cached=257, kv_heads=8, head_dim=128, kv="fp8",
             block_size=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_HEADS = ((14, 2, 64), (32, 8, 128), (64, 8, 128), (16, 8, 256))


def draw(rng):
    op = rng.choice(("indices", "masks", "mrope", "attend", "attend", "accept"))
    if op == "indices":
        return dict(op=op, batch=_log(rng, 1, 512), new=_log(rng, 1, 300), ragged=rng.uniform(0, 1), cached=_log(rng, 1, 9000),
                    block_size=rng.choice((16, 32, 64, 128)), pad=rng.randrange(0, 64))
    if op == "masks":
        return dict(op=op, batch=_log(rng, 1, 192), nodes=_log(rng, 1, 300), ragged=rng.uniform(0, 0.9))
    if op == "mrope":
        hq, hkv, d = rng.choice(_HEADS)
        return dict(op=op, tokens=_log(rng, 1, 4000), q_heads=hq, kv_heads=hkv, head_dim=d, dtype=rng.choice(("bf16", "fp16", "fp32")),
                    norm=rng.random() < 0.5, block_size=rng.choice((16, 32, 128)), axes=rng.choice((2, 3, 4)),
                    dealt=rng.random() < 0.5)
    if op == "accept":
        _, hkv, d = rng.choice(_HEADS)
        nodes = _log(rng, 1, 61)
        return dict(op=op, batch=_log(rng, 1, 256), path=rng.randrange(1, min(nodes, 13) + 1), nodes=nodes, cached=_log(rng, 1, 500),
                    kv_heads=hkv, head_dim=d, kv=rng.choice(("bf16", "fp16", "fp32", "int8", "fp8")), block_size=rng.choice((16, 32, 128)))
    hq, hkv, d = rng.choice(_HEADS)
    q = rng.choice(("bf16", "bf16", "fp16"))
    c = dict(op=op, batch=_log(rng, 1, 128), nodes=_log(rng, 1, 64), len=_log(rng, 64, 32768), q_heads=hq, kv_heads=hkv, head_dim=d,
             q=q, kv=rng.choice((q, "int8", "fp8")), block_size=rng.choice((32, 64, 128)), ragged=rng.uniform(0, 0.9))
    most = work(listed()[9])
    while work(c)["bytes"] > 2 ** 30 or work(c)["flops"] > most["flops"]:
        c["len"] = max(c["nodes"], c["len"] * 3 // 4)
        c["batch"] = max(1, c["batch"] * 3 // 4)
    return c


def _spread(count, top, ragged, least=0):
    """`count` whole numbers from `top` down to about (1 - ragged) * top, in no order: the same ones for every seed."""
    return [max(least, int(round(top * (1.0 - ragged * ((b * _GOLDEN) % 1.0))))) for b in range(count)]


def _attend_sizes(c):
    n = _spread(c["batch"], c["nodes"], min(c["ragged"], 0.5), 1)
    lens = [max(a, b) for a, b in zip(_spread(c["batch"], c["len"], c["ragged"], 1), n)]
    return n, lens


def work(c):
    op = c["op"]
    if op == "indices":
        new = _spread(c["batch"], c["new"], c["ragged"], 1)
        cached = _spread(c["batch"], c["cached"], c["ragged"], 0)
        blocks = sum(-(-(a + b) // c["block_size"]) for a, b in zip(new, cached))
        # lengths, request ids, held in; three arrays out; block lists in, table and compact list out; slots, positions
        return dict(bytes=4 * 9 * c["batch"] + 3 * 4 * blocks + 12 * (sum(new) + c["pad"]), flops=0)
    if op == "masks":
        t = sum(_spread(c["batch"], c["nodes"], c["ragged"], 1))
        return dict(bytes=t * (4 + 8 * -(-c["nodes"] // 64) + 8) + 12 * c["batch"], flops=0)
    if op == "mrope":
        eb, t, d = _BYTES[c["dtype"]], c["tokens"], c["head_dim"]
        qk, v = c["q_heads"] + c["kv_heads"], c["kv_heads"]
        return dict(bytes=t * d * eb * (qk + v) + t * d * eb * (qk + 2 * v) + t * (4 * d + 8 * c["axes"] + 4), flops=t * qk * d * (7 if c["norm"] else 3))
    if op == "accept":
        row = c["kv_heads"] * (c["head_dim"] * _BYTES[c["kv"]] + (4 if c["kv"] in ("int8", "fp8") else 0))
        return dict(bytes=c["batch"] * (c["path"] * (4 * row + 12) + 16), flops=0)
    n, lens = _attend_sizes(c)
    row = c["kv_heads"] * (c["head_dim"] * _BYTES[c["kv"]] + (4 if c["kv"] in ("int8", "fp8") else 0))
    qo = sum(n) * c["q_heads"] * (2 * c["head_dim"] * _BYTES[c["q"]] + 4)
    return dict(bytes=2 * row * sum(lens) + qo + sum(n) * 8 + 4 * sum(-(-x // c["block_size"]) for x in lens),
                flops=4.0 * c["q_heads"] * c["head_dim"] * sum(a * b for a, b in zip(n, lens)))


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _indptr(counts):
    total, at = 0, [0]
    for n in counts:
        total += n
        at.append(total)
    return _i32(at)


def _parents(gen, counts):
    """A random tree per sequence: node 0 a child of the context, node j of one of the nodes before it."""
    j = torch.cat([torch.arange(n, device=DEVICE) for n in counts])
    r = torch.rand(j.numel(), generator=gen, device=DEVICE)
    return torch.minimum((r * j).floor().long(), j - 1).to(torch.int32)


def _tables(gen, lens, block_size, spare=0):
    """Shuffled disjoint block lists; block 0 is nobody's."""
    need = [-(-n // block_size) for n in lens]
    ids = (torch.randperm(sum(need) + spare, generator=gen, device=DEVICE) + 1).to(torch.int32)
    width = max(max(need), 1)
    col = torch.arange(width, device=DEVICE)
    n = torch.tensor(need, device=DEVICE)
    at = torch.cumsum(n, 0) - n
    held = col[None] < n[:, None]
    table = torch.where(held, ids[torch.where(held, at[:, None] + col[None], 0)], 0)
    return table.to(torch.int32).contiguous(), sum(need) + spare + 1, ids[sum(need):].contiguous()


def _cache(gen, kv, shape):
    dt = _DTYPES[kv]
    if kv == "int8":
        make = lambda: torch.randint(-127, 128, shape, generator=gen, device=DEVICE, dtype=torch.int8)  # noqa: E731
    else:
        make = lambda: torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dt)  # noqa: E731
    k, v = make(), make()
    if kv not in ("int8", "fp8"):
        return k, v, None, None
    unit = 1.0 / 64.0 if kv == "int8" else 1.0
    scales = [(torch.rand(shape[:3], generator=gen, device=DEVICE) + 0.5) * unit for _ in range(2)]
    return k, v, scales[0], scales[1]


def _cos_sin(max_position, rotary_dim):
    inv = 10000.0 ** (-torch.arange(0, rotary_dim, 2, device=DEVICE, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(max_position, device=DEVICE, dtype=torch.float64)[:, None] * inv[None]
    return torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()


def _sections(axes, half):
    """How many of a head's rotation pairs each axis turns: even parts, what is left over to the first axis."""
    part = [half // axes] * axes
    part[0] += half - sum(part)
    return tuple(part)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed) * 7 + 3)
    s = {"case": c}
    op = c["op"]
    if op == "indices":
        B, bs = c["batch"], c["block_size"]
        new = _spread(B, c["new"], c["ragged"], 1)
        cached = _spread(B, c["cached"], c["ragged"], 0)
        need = [-(-(a + b) // bs) for a, b in zip(new, cached)]
        rows = B + 5
        order = torch.randperm(rows, generator=gen, device=DEVICE)[:B].to(torch.int32)
        table, blocks, free = _tables(gen, cached, bs, spare=sum(need) + 7)
        width = max(need)
        pool = torch.zeros(rows, width, dtype=torch.int32, device=DEVICE)
        pool[order.long(), :table.size(1)] = table
        total = sum(new) + c["pad"]
        empty = lambda *n, dt=torch.int32: torch.zeros(*n, dtype=dt, device=DEVICE)  # noqa: E731
        s.update(cached=_i32(cached), new=_i32(new), held=_i32([-(-a // bs) for a in cached]), order=order, pool=pool, free=free,
                 head=_i32([3]), table=empty(B, width), seq_lens=empty(B), q_indptr=empty(B + 1), slots=empty(total),
                 positions=empty(total, dt=torch.int64), kv_indptr=empty(B + 1), kv_indices=empty(sum(need)), last=empty(B),
                 held_out=empty(B), head_out=empty(2))
        return s
    if op == "masks":
        counts = _spread(c["batch"], c["nodes"], c["ragged"], 1)
        t = sum(counts)
        s.update(parents=_parents(gen, counts), q_indptr=_indptr(counts),
                 base=torch.randint(0, 9000, (c["batch"],), generator=gen, device=DEVICE, dtype=torch.int32),
                 mask=torch.zeros(t, -(-c["nodes"] // 64), dtype=torch.int64, device=DEVICE),
                 positions=torch.zeros(t, dtype=torch.int64, device=DEVICE))
        return s
    if op == "mrope":
        t, hq, hkv, d, dt = c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"], _DTYPES[c["dtype"]]
        bs = c["block_size"]
        blocks = -(-t // bs) + 2
        s.update(qkv=torch.randn(t, (hq + 2 * hkv) * d, generator=gen, device=DEVICE).to(dt),
                 cos_sin=_cos_sin(8192, d), positions=torch.randint(0, 8192, (c["axes"], t), generator=gen, device=DEVICE),
                 sections=_sections(c["axes"], d // 2),
                 slots=torch.randperm(blocks * bs, generator=gen, device=DEVICE)[:t].to(torch.int32),
                 k_cache=torch.zeros(blocks, hkv, bs, d, dtype=dt, device=DEVICE),
                 v_cache=torch.zeros(blocks, hkv, bs, d, dtype=dt, device=DEVICE))
        s["q_weight"] = s["k_weight"] = None
        if c["norm"]:
            s["q_weight"] = (torch.rand(d, generator=gen, device=DEVICE) + 0.5).to(dt)
            s["k_weight"] = (torch.rand(d, generator=gen, device=DEVICE) + 0.5).to(dt)
        return s
    if op == "accept":
        lens = [x + c["nodes"] for x in _spread(c["batch"], c["cached"], 0.5, 0)]
        table, blocks, _ = _tables(gen, lens, c["block_size"])
        k, v, ks, vs = _cache(gen, c["kv"], (blocks, c["kv_heads"], c["block_size"], c["head_dim"]))
        pick = torch.rand(c["batch"], c["nodes"], generator=gen, device=DEVICE).argsort(1)[:, :c["path"]].sort(1).values
        s.update(k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, table=table, cached=_i32([x - c["nodes"] for x in lens]),
                 accepted=pick.to(torch.int32).contiguous(),
                 count=torch.randint(0, c["path"] + 1, (c["batch"],), generator=gen, device=DEVICE, dtype=torch.int32),
                 new_lens=torch.zeros(c["batch"], dtype=torch.int32, device=DEVICE))
        return s
    n, lens = _attend_sizes(c)
    table, blocks, _ = _tables(gen, lens, c["block_size"])
    k, v, ks, vs = _cache(gen, c["kv"], (blocks, c["kv_heads"], c["block_size"], c["head_dim"]))
    t = sum(n)
    q = torch.randn(t, c["q_heads"], c["head_dim"], generator=gen, device=DEVICE).to(_DTYPES[c["q"]])
    indptr = _indptr(n)
    s.update(q=q, k_cache=k, v_cache=v, k_scale=ks, v_scale=vs, table=table, seq_lens=_i32(lens), q_indptr=indptr, nodes=max(n),
             max_len=max(lens), total_len=sum(lens), scale=1.0 / math.sqrt(c["head_dim"]),
             mask=_plain_masks(_parents(gen, n), indptr, max(n))[0], out=torch.empty_like(q),
             lse=torch.empty(t, c["q_heads"], dtype=torch.float32, device=DEVICE))
    return s


# ---------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------

def _sequence_of(q_indptr, tokens):
    t = torch.arange(tokens, device=q_indptr.device)
    b = torch.searchsorted(q_indptr.long(), t, right=True) - 1
    return b, t - q_indptr.long()[b]


def _plain_indices(s):
    bs = s["case"]["block_size"]
    cached, new, held = s["cached"].long(), s["new"].long(), s["held"].long()
    req, pool, free = s["order"].long(), s["pool"], s["free"]
    lens = cached + new
    need = (lens + bs - 1) // bs
    grow = (need - held).clamp(min=0)
    first = s["head"].long() + torch.cumsum(grow, 0) - grow
    col = torch.arange(pool.size(1), device=pool.device)[None]
    fresh = (col >= held[:, None]) & (col < need[:, None])
    taken = free[(first[:, None] + col - held[:, None]).clamp(0, free.numel() - 1)]
    rows = torch.where(fresh, taken, pool[req])
    pool[req] = rows
    inside = col < need[:, None]
    table = torch.where(inside, rows, 0)
    q_indptr = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    kv_indptr = torch.cat([torch.zeros_like(need[:1]), torch.cumsum(need, 0)])
    indices = rows[inside]
    total = s["slots"].numel()
    b, j = _sequence_of(q_indptr[:-1], total)
    live = torch.arange(total, device=pool.device) < q_indptr[-1]
    pos = cached[b] + j
    slots = rows[b, torch.where(live, pos // bs, 0)].long() * bs + pos % bs
    as32 = lambda x: x.to(torch.int32)  # noqa: E731
    return {"table": table, "seq_lens": as32(lens), "q_indptr": as32(q_indptr), "slots": as32(torch.where(live, slots, -1)),
            "positions": torch.where(live, pos, 0), "kv_indptr": as32(kv_indptr), "kv_indices": indices,
            "last": as32(torch.where(lens > 0, (lens - 1) % bs + 1, 0)), "held": as32(torch.maximum(held, need)),
            "head": as32(torch.cat([s["head"].long() + grow.sum(), torch.zeros_like(new[:1])])), "pool": pool}


def _plain_masks(parents, q_indptr, most):
    t = parents.numel()
    b, j = _sequence_of(q_indptr[:-1], t)
    words = -(-most // 64)
    up = torch.where(parents >= 0, q_indptr.long()[b] + parents.long(), t)
    up = torch.cat([up, up.new_full((1,), t)])
    seen = torch.zeros(t + 1, words * 64, dtype=torch.bool, device=parents.device)
    seen[torch.arange(t, device=parents.device), j] = True
    for _ in range(max(1, math.ceil(math.log2(max(most, 2))))):  # ancestors within 1, 2, 4, ... steps
        seen = seen | seen[up]
        up = up[up]
    seen = seen[:t]
    bit = torch.arange(64, device=parents.device)
    return (seen.view(t, words, 64).long() << bit).sum(-1), seen.sum(1) - 1, b


def _axis_of_pair(sections, dealt, device):
    half = sum(sections)
    if not dealt:
        return torch.repeat_interleave(torch.arange(len(sections), device=device), torch.tensor(sections, device=device))
    j = torch.arange(half, device=device)
    a = j % len(sections)
    return torch.where(j // len(sections) < torch.tensor(sections, device=device)[a], a, 0)


def _rotated(x, c, cos, sin, weight, eps):
    """x [T, H, D] in the arithmetic's type: norm, then the pairs (j, j + D/2) turned."""
    if weight is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * weight
    lo, hi = x.chunk(2, -1)
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def _plain_mrope(s):
    c = s["case"]
    hq, hkv, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    qkv = s["qkv"]
    t = qkv.size(0)
    x = qkv.view(t, hq + 2 * hkv, d).float()
    pair = torch.arange(d // 2, device=qkv.device)
    at = s["positions"][_axis_of_pair(s["sections"], c["dealt"], qkv.device)].t()
    cos, sin = s["cos_sin"][at, pair][:, None], s["cos_sin"][at, pair + d // 2][:, None]
    wq, wk = (w.float() if w is not None else None for w in (s["q_weight"], s["k_weight"]))
    q = _rotated(x[:, :hq], c, cos, sin, wq, 1e-6)
    k = _rotated(x[:, hq:hq + hkv], c, cos, sin, wk, 1e-6)
    qkv.view(t, hq + 2 * hkv, d)[:, :hq + hkv] = torch.cat([q, k], 1).to(qkv.dtype)
    slot, bs = s["slots"].long(), c["block_size"]
    rows = qkv.view(t, hq + 2 * hkv, d)
    s["k_cache"][slot // bs, :, slot % bs] = rows[:, hq:hq + hkv]
    s["v_cache"][slot // bs, :, slot % bs] = rows[:, hq + hkv:]
    return {"qkv": qkv, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _plain_attend(s):
    c = s["case"]
    hkv, d, bs = c["kv_heads"], c["head_dim"], c["block_size"]
    g = c["q_heads"] // hkv
    q, table, mask, indptr = s["q"], s["table"].long(), s["mask"], s["q_indptr"].long()
    lens, n, most = s["seq_lens"].long(), indptr[1:] - indptr[:-1], s["nodes"]
    B, t, L = lens.numel(), q.size(0), s["max_len"]
    pos = torch.arange(L, device=q.device)
    blk, slot = table[:, pos // bs], pos % bs
    k, v = s["k_cache"][blk, :, slot].float(), s["v_cache"][blk, :, slot].float()  # [B, L, Hkv, D]
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][blk, :, slot][..., None], v * s["v_scale"][blk, :, slot][..., None]
    row = (indptr[:-1, None] + torch.arange(most, device=q.device)).clamp(max=t - 1)
    qp = q[row].float().view(B, most, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(B * hkv, most * g, d)
    u = pos[None] - (lens - n)[:, None]                                            # the key's place in the tree
    words = mask[row].gather(2, (u.clamp(0, mask.size(1) * 64 - 1) >> 6)[:, None].expand(B, most, L))
    bit = (words >> (u & 63)[:, None]) & 1
    sees = ((u < 0)[:, None] | (bit == 1)) & (pos[None] < lens[:, None])[:, None]  # [B, n, L]
    x = torch.bmm(qp, k.permute(0, 2, 3, 1).reshape(B * hkv, d, L).contiguous()) * s["scale"]
    x = x.view(B, hkv, most, g, L).masked_fill(~sees[:, None, :, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    total = e.sum(-1, keepdim=True)
    o = torch.bmm(e.view(B * hkv, most * g, L), v.permute(0, 2, 1, 3).reshape(B * hkv, L, d).contiguous())
    o = o.view(B, hkv, most, g, d) / torch.where(total > 0, total, 1.0)
    lse = ((m + total.log()) / math.log(2.0)).squeeze(-1)
    b, j = _sequence_of(indptr[:-1], t)
    return {"out": o[b, :, j].reshape(t, hkv * g, d).to(q.dtype), "lse": lse[b, :, j].reshape(t, hkv * g)}


def _plain_accept(s):
    bs = s["case"]["block_size"]
    cached, table, path = s["cached"].long(), s["table"].long(), s["accepted"].long()
    i = torch.arange(path.size(1), device=path.device)[None].expand_as(path)
    live = i < s["count"].long()[:, None]
    b = torch.arange(path.size(0), device=path.device)[:, None].expand_as(path)[live]
    src, dst = (cached[:, None] + path)[live], (cached[:, None] + i)[live]
    from_block, to_block = table[b, src // bs], table[b, dst // bs]
    as_bytes = lambda x: x.view(torch.uint8) if x.element_size() == 1 else x  # noqa: E731
    k, v = as_bytes(s["k_cache"]), as_bytes(s["v_cache"])
    k[to_block, :, dst % bs] = k[from_block, :, src % bs]
    v[to_block, :, dst % bs] = v[from_block, :, src % bs]
    out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "lens": (cached + s["count"].long()).to(torch.int32)}
    if s["k_scale"] is not None:
        ks, vs = s["k_scale"], s["v_scale"]
        ks[to_block, :, dst % bs] = ks[from_block, :, src % bs]
        vs[to_block, :, dst % bs] = vs[from_block, :, src % bs]
        out.update(k_scale=ks, v_scale=vs)
    return out


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        if op == "indices":
            return _plain_indices(s)
        if op == "masks":
            mask, depth, b = _plain_masks(s["parents"], s["q_indptr"], c["nodes"])
            return {"mask": mask, "positions": s["base"].long()[b] + depth}
        if op == "mrope":
            return _plain_mrope(s)
        if op == "attend":
            return _plain_attend(s)
        return _plain_accept(s)
    from xllm_wxh_amd import ops
    if op == "indices":
        ops.build_step_indices(s["cached"], s["pool"], c["block_size"], s["table"], s["seq_lens"], s["q_indptr"], s["slots"],
                               s["positions"], new_lens=s["new"], request_ids=s["order"], held_blocks=s["held"],
                               free_blocks=s["free"], free_head=s["head"], held_blocks_out=s["held_out"],
                               free_head_out=s["head_out"], paged_kv_indptr=s["kv_indptr"], paged_kv_indices=s["kv_indices"],
                               paged_kv_last_page_len=s["last"])
        return {"table": s["table"], "seq_lens": s["seq_lens"], "q_indptr": s["q_indptr"], "slots": s["slots"],
                "positions": s["positions"], "kv_indptr": s["kv_indptr"], "kv_indices": s["kv_indices"], "last": s["last"],
                "held": s["held_out"], "head": s["head_out"], "pool": s["pool"]}
    if op == "masks":
        ops.tree_masks(s["parents"], s["mask"], s["positions"], s["base"], q_indptr=s["q_indptr"])
        return {"mask": s["mask"], "positions": s["positions"]}
    if op == "mrope":
        ops.mrope_kv_write(s["qkv"], c["q_heads"], c["kv_heads"], c["head_dim"], s["cos_sin"], s["positions"], s["sections"],
                           s["k_cache"], s["v_cache"], s["slots"], mrope_interleaved=c["dealt"], q_weight=s["q_weight"],
                           k_weight=s["k_weight"], eps=1e-6)
        return {"qkv": s["qkv"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if op == "attend":
        ops.batch_tree_decode(s["q"], s["k_cache"], s["v_cache"], s["out"], s["table"], s["seq_lens"], s["mask"],
                              q_indptr=s["q_indptr"], q_per_seq=s["nodes"], scale=s["scale"], output_lse=s["lse"],
                              k_cache_quant_scale=s["k_scale"], v_cache_quant_scale=s["v_scale"], max_seq_len=s["max_len"],
                              total_kv_len=s["total_len"])
        return {"out": s["out"], "lse": s["lse"]}
    ops.move_accepted_tokens(s["k_cache"], s["v_cache"], s["table"], s["cached"], s["accepted"], s["count"], s["new_lens"],
                             k_cache_scale=s["k_scale"], v_cache_scale=s["v_scale"])
    out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"], "lens": s["new_lens"]}
    if s["k_scale"] is not None:
        out.update(k_scale=s["k_scale"], v_scale=s["v_scale"])
    return out


# ---------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------

def exact(case, seed):
    """What run returns, from the operators' definitions in 64 bits: sequence by sequence, head by head.  Index
    arrays, masks and moved rows are whole numbers or copies, which have no closer value."""
    if case["op"] == "mrope":
        return _exact_mrope(prepare(case, seed))
    if case["op"] == "attend":
        return _exact_attend(prepare(case, seed))
    return None


def _exact_mrope(s):
    c = s["case"]
    hq, hkv, d, bs = c["q_heads"], c["kv_heads"], c["head_dim"], c["block_size"]
    half, sec = d // 2, s["sections"]
    x = s["qkv"].double().view(c["tokens"], hq + 2 * hkv, d).clone()
    axis = []
    for a, n in enumerate(sec):
        axis += [a] * n
    if c["dealt"]:
        axis = [j % len(sec) if j // len(sec) < sec[j % len(sec)] else 0 for j in range(half)]
    for heads, w in ((slice(0, hq), s["q_weight"]), (slice(hq, hq + hkv), s["k_weight"])):
        part = x[:, heads]
        if w is not None:
            part = part / torch.sqrt((part * part).sum(-1, keepdim=True) / d + 1e-6) * w.double()
        turned = part.clone()
        for j in range(half):
            row = s["cos_sin"][s["positions"][axis[j]]].double()
            cos, sin = row[:, j, None], row[:, half + j, None]
            turned[:, :, j] = part[:, :, j] * cos - part[:, :, half + j] * sin
            turned[:, :, half + j] = part[:, :, half + j] * cos + part[:, :, j] * sin
        x[:, heads] = turned
    k, v = s["k_cache"].double(), s["v_cache"].double()
    slot = s["slots"].long()
    k[slot // bs, :, slot % bs] = x[:, hq:hq + hkv]
    v[slot // bs, :, slot % bs] = x[:, hq + hkv:]
    return {"qkv": x.reshape(c["tokens"], -1), "k_cache": k, "v_cache": v}


def _exact_attend(s):
    c = s["case"]
    hkv, d, bs = c["kv_heads"], c["head_dim"], c["block_size"]
    g = c["q_heads"] // hkv
    out, lse = s["q"].double().clone(), s["lse"].double().clone()
    starts, lens = s["q_indptr"].tolist(), s["seq_lens"].tolist()
    for b, length in enumerate(lens):
        n = starts[b + 1] - starts[b]
        blocks = s["table"][b, :-(-length // bs)].long()
        rows = slice(starts[b], starts[b + 1])
        bits = (s["mask"][rows][:, :, None] >> torch.arange(64, device=DEVICE)) & 1
        sees = torch.ones(n, length, dtype=torch.bool, device=DEVICE)
        sees[:, length - n:] = bits.reshape(n, -1)[:, :n] == 1
        for h in range(hkv):
            k = s["k_cache"][blocks, h].double().reshape(-1, d)[:length]
            v = s["v_cache"][blocks, h].double().reshape(-1, d)[:length]
            if s["k_scale"] is not None:
                k = k * s["k_scale"][blocks, h].double().reshape(-1, 1)[:length]
                v = v * s["v_scale"][blocks, h].double().reshape(-1, 1)[:length]
            q = s["q"][rows, h * g:(h + 1) * g].double().reshape(n * g, d)
            x = (q @ k.t().contiguous() * s["scale"]).view(n, g, length)
            x = x.masked_fill(~sees[:, None], -math.inf)
            top = torch.logsumexp(x, -1, keepdim=True)
            out[rows, h * g:(h + 1) * g] = (torch.exp(x - top).view(n * g, length) @ v).view(n, g, d)
            lse[rows, h * g:(h + 1) * g] = top.squeeze(-1) / math.log(2.0)
    return {"out": out, "lse": lse}
