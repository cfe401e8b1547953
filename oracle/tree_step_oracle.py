"""CPU restatement, in 64 bits and index by index, of a speculative step over a tree of drafted tokens: the index
arrays from request lengths, ancestor masks, the multi-axis rotary embedding, attention under the masks, and the move
of the accepted rows.  Test infrastructure only; written from the definitions in include/xllm_hip_paged_kv.h, with no
code of the device side."""
import math

import numpy as np


def step_indices(cached, new, request_ids, held, pool, free, head, block_size, table_width, num_rows, kv_capacity=None):
    """Returns a dict of the arrays; `pool` is updated in place.  held None: the rows of pool hold everything."""
    B = len(cached)
    width = min(pool.shape[1], table_width)
    table = np.zeros((B, table_width), np.int64)
    seq_lens, q_indptr, held_out = np.zeros(B, np.int64), np.zeros(B + 1, np.int64), np.zeros(B, np.int64)
    kv_indptr, last, kv = np.zeros(B + 1, np.int64), np.zeros(B, np.int64), []
    slots, positions = np.full(num_rows, -1, np.int64), np.zeros(num_rows, np.int64)
    at, missing, row = head or 0, 0, 0
    for b in range(B):
        c, n, r = max(int(cached[b]), 0), max(int(new[b]), 0), int(request_ids[b])
        need = -(-(c + n) // block_size)
        ok = 0 <= r < pool.shape[0]
        mine = [] if not ok else [int(x) for x in pool[r, :(pool.shape[1] if held is None else min(max(int(held[b]), 0), pool.shape[1]))]]
        held_out[b] = len(mine)
        while ok and free is not None and len(mine) < min(need, width):
            if at >= len(free):
                break
            pool[r, len(mine)] = free[at]
            mine.append(int(free[at]))
            at += 1
        held_out[b] = max(held_out[b], len(mine))
        mine = mine[:min(need, width)]
        missing += need - len(mine)
        table[b, :len(mine)] = mine
        listed = min(need, table_width)
        kv += [int(table[b, i]) for i in range(listed)]
        kv_indptr[b + 1] = kv_indptr[b] + listed
        last[b] = 0 if need == 0 else (block_size if need > table_width else (c + n - 1) % block_size + 1)
        seq_lens[b], q_indptr[b + 1] = c + n, q_indptr[b] + n
        for j in range(n):
            if row < num_rows:
                pos = c + j
                positions[row] = pos
                i = pos // block_size
                if i < len(mine) and mine[i] >= 0 and mine[i] * block_size + pos % block_size < 2 ** 31:
                    slots[row] = mine[i] * block_size + pos % block_size
            row += 1
    return dict(block_table=table, seq_lens=seq_lens, q_indptr=q_indptr, slot_mapping=slots, positions=positions,
                paged_kv_indptr=kv_indptr, paged_kv_indices=np.array(kv[:kv_capacity], np.int64), paged_kv_last_page_len=last,
                held_blocks_out=held_out, free_head_out=np.array([at, missing]))


def tree_masks(parents, q_indptr, base, words):
    """mask [rows, words] (uint64) and positions [rows]; rows of no sequence are 0 / 0."""
    mask, positions = np.zeros((len(parents), words), np.uint64), np.zeros(len(parents), np.int64)
    for b in range(len(q_indptr) - 1):
        lo, hi = int(q_indptr[b]), int(q_indptr[b + 1])
        limit = min(hi - lo, 64 * words)
        for v in range(hi - lo):
            seen, at = [], v
            while v < limit and 0 <= at < limit and at not in seen:
                seen.append(at)
                at = int(parents[lo + at])
            for u in seen:
                mask[lo + v, u // 64] |= np.uint64(1) << np.uint64(u % 64)
            positions[lo + v] = (0 if base is None else int(base[b])) + max(len(seen) - 1, 0)
    return mask, positions


def axis_of_pairs(sections, dealt):
    if not dealt:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    k = len(sections)
    return [j % k if j // k < sections[j % k] else 0 for j in range(sum(sections))]


def mrope(x, positions, table, sections, dealt, interleave, weight=None, eps=1e-6):
    """x [tokens, heads, head_dim]: norm (optional), then the pairs of the first table.shape[1] elements turned."""
    x = np.asarray(x, np.float64).copy()
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    half = table.shape[1] // 2
    out = x.copy()
    for j, a in enumerate(axis_of_pairs(sections, dealt)):
        row = np.clip(positions[a], 0, table.shape[0] - 1)
        c, s = table[row, j][:, None], table[row, half + j][:, None]
        p, q = (2 * j, 2 * j + 1) if interleave else (j, j + half)
        out[:, :, p] = x[:, :, p] * c - x[:, :, q] * s
        out[:, :, q] = x[:, :, q] * c + x[:, :, p] * s
    return out


def tree_attention(q, k_rows, v_rows, q_indptr, lens, mask, scale):
    """q [rows, Hq, D]; k_rows / v_rows: per sequence [len, Hkv, D]; mask [rows, words] uint64.
    Returns out, lse (base 2), and what error bounds are made of: sum_t p_t |v_t| [rows, Hq, D] and the largest
    sum_d |q_d k_d| * scale and sum_d |k_d| * scale over the keys a row sees [rows, Hq]."""
    rows, Hq, D = q.shape
    out, absv = np.zeros((rows, Hq, D)), np.zeros((rows, Hq, D))
    lse, dots, ks = np.full((rows, Hq), -math.inf), np.zeros((rows, Hq)), np.zeros((rows, Hq))
    for b in range(len(lens)):
        lo, n, L = int(q_indptr[b]), int(q_indptr[b + 1] - q_indptr[b]), int(lens[b])
        Hkv = k_rows[b].shape[1]
        g = Hq // Hkv
        for j in range(n):
            sees = np.zeros(L, bool)
            for t in range(L):
                u = t - (L - n)
                sees[t] = u < 0 or (u // 64 < mask.shape[1] and (int(mask[lo + j, u // 64]) >> (u % 64)) & 1 == 1)
            idx = np.nonzero(sees)[0]
            if len(idx) == 0:
                continue
            for h in range(Hq):
                kk, vv = k_rows[b][idx, h // g].astype(np.float64), v_rows[b][idx, h // g].astype(np.float64)
                qq = q[lo + j, h].astype(np.float64)
                x = kk @ qq * scale
                m = x.max()
                e = np.exp(x - m)
                out[lo + j, h] = e @ vv / e.sum()
                absv[lo + j, h] = e @ np.abs(vv) / e.sum()
                lse[lo + j, h] = (m + math.log(e.sum())) / math.log(2.0)
                dots[lo + j, h] = (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
                ks[lo + j, h] = np.abs(kk).sum(1).max() * abs(scale)
    return out, lse, absv, dots, ks


def move_accepted(rows_of, set_row, cached, accepted, count, width, capacity):
    """rows_of(b, token) -> a copy of the token's rows or None; set_row(b, token, rows).  Every sequence's rows are
    read before any is written."""
    for b in range(len(cached)):
        got = []
        for i in range(min(max(int(count[b]), 0), width)):
            src, dst = int(cached[b]) + int(accepted[b][i]), int(cached[b]) + i
            if accepted[b][i] < 0 or not (0 <= src < capacity and 0 <= dst < capacity):
                continue
            r = rows_of(b, src)
            if r is not None and rows_of(b, dst) is not None:
                got.append((dst, r))
        for dst, r in got:
            set_row(b, dst, r)
