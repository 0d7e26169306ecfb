"""CPU restatement, in 64 bits, of one step of speculative decoding over the paged cache (the parity oracle for
pa_draft_layout, pa_draft_attention, pa_verify_drafts and pa_draft_commit).

TEST INFRASTRUCTURE ONLY.  Nothing under the product package imports this module.  Everything is written row by row
and node by node, from the definitions; the reference's own verification (src/inference/speculative.py) covers greedy
and sampled chains without top-p, a special case of `verify`.

Pinning (tests/test_drafts_host.py): over an exhaustive grid of uniform numbers `verify` emits tokens with exactly the
target's probabilities, for chains with and without draft probabilities and for trees; greedy chains reproduce the
reference's rule (longest prefix equal to the argmax, then the argmax).
"""
import math

import torch


def ancestors(parents):
    """Per node the set of the node and its ancestors; a parent outside [0, i) makes node i a root."""
    sets = []
    for i, p in enumerate(parents):
        sets.append({i} | (sets[p] if 0 <= p < i else set()))
    return sets


def layout(parents, base, real, table, block_size, num_blocks):
    """(positions, slots, list of ancestor sets) of one row."""
    sets = ancestors(parents)
    positions, slots = [], []
    for i, s in enumerate(sets):
        if i >= real:
            positions.append(0)
            slots.append(-1)
            continue
        positions.append(base + len(s) - 1)
        col = (base + i) // block_size
        block = table[col] if col < len(table) else -1
        slots.append(block * block_size + (base + i) % block_size if 0 <= block < num_blocks else -1)
    return positions, slots, sets


def mask_words(sets, nodes):
    """int64 [nodes, words] of ancestor sets."""
    words = (nodes + 63) // 64
    out = torch.zeros(nodes, words, dtype=torch.int64)
    for i, s in enumerate(sets):
        for w in range(words):
            v = sum(1 << (j % 64) for j in s if j // 64 == w)
            out[i, w] = v - (1 << 64) if v >= 1 << 63 else v
    return out


def row_kv(cache, scale, table, count, block_size):
    """fp64 [count, kv_heads, head_dim] of one row's first `count` tokens."""
    pos = torch.arange(count)
    ids = torch.as_tensor(table, dtype=torch.long)[pos // block_size]
    x = cache[ids, pos % block_size].double()
    return x if scale is None else x / scale[ids, pos % block_size].double()[:, None, None]


def attention(q, k, v, base, sets, real, scale):
    """One row: q [nodes, heads, dim]; k, v fp64 [base + real, kv_heads, dim]; sets: the nodes each node sees.
    Returns (out, spread, weight): out [nodes, heads, dim], spread = sum_j p_j |v_j| (what a relative error of the
    probabilities can move), weight = sum_j |v_j| over the visible keys (what an absolute one can)."""
    nodes, heads, dim = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(nodes, heads, dim, dtype=torch.float64)
    spread, weight = torch.zeros_like(out), torch.zeros_like(out)
    for i in range(real):
        see = list(range(base)) + [base + j for j in sorted(sets[i]) if j < real]
        if not see:
            continue
        for h in range(heads):
            s = (k[see, h // group] @ q[i, h].double()) * scale
            p = torch.softmax(s, 0)
            out[i, h] = p @ v[see, h // group]
            spread[i, h] = p @ v[see, h // group].abs()
            weight[i, h] = v[see, h // group].abs().sum(0)
    return out, spread, weight


def weights(logits, temperature, top_p):
    """fp64 weights of one row: exp((l - max) / T), zero outside the nucleus (a token stays while the mass of the
    strictly likelier ones is at most top_p of all); NaN and -inf weigh nothing."""
    l = logits.double()
    l = torch.where(torch.isnan(l), torch.full_like(l, -math.inf), l)
    top = l.max()
    if top == -math.inf:
        return torch.zeros_like(l)
    w = torch.where(l == top, torch.ones_like(l), torch.exp((l - top) / temperature))
    if top_p < 1:
        down, order = torch.sort(w, descending=True)
        upto = down.cumsum(0)
        above, start = torch.zeros_like(down), 0.0
        for i in range(len(down)):
            if i and down[i] != down[i - 1]:
                start = float(upto[i - 1])
            above[i] = start
        keep = above <= top_p * upto[-1]
        w = torch.zeros_like(w)
        w[order[keep]] = down[keep]
    return w


def draw(w, u):
    """First index whose running sum exceeds u times the total; the last positive entry by rounding, 0 without any."""
    upto = w.cumsum(0)
    hit = torch.nonzero(upto > u * upto[-1]).flatten()
    if len(hit):
        return int(hit[0])
    some = torch.nonzero(w > 0).flatten()
    return int(some[-1]) if len(some) else 0


def first_max(logits):
    l = torch.where(torch.isnan(logits.double()), torch.full_like(logits.double(), -math.inf), logits.double())
    return int(torch.nonzero(l == l.max()).flatten()[0]) if l.max() > -math.inf else 0


def verify(logits, tokens, u, parents, real, temperature, top_p, probs=None):
    """One row: (emitted tokens, kept nodes).  logits [nodes, vocab]; probs [nodes - 1, vocab] or None."""
    if real == 0:
        return [], []
    vocab = logits.shape[1]
    node, path, emitted = 0, [0], []
    while True:
        children = [c for c in range(1, real) if parents[c] == node]
        if temperature <= 0:
            best = first_max(logits[node])
            taken = next((c for c in children if int(tokens[c]) == best), None)
            rest = None
        else:
            w = weights(logits[node], temperature, top_p)
            rest, taken = w.clone(), None
            for c in children:
                t = int(tokens[c])
                if probs is None:
                    good = 0 <= t < vocab and float(u[c]) * float(rest.sum()) < float(rest[t])
                else:
                    good = 0 <= t < vocab and float(u[c]) * float(probs[node, t]) * float(w.sum()) < float(w[t])
                if good:
                    taken = c
                    break
                if probs is None and 0 <= t < vocab:
                    rest[t] = 0.0
            if taken is None and children and probs is not None:
                rest = (w / w.sum() - probs[node].double()).clamp(min=0)
            if rest.sum() <= 0:
                rest = w
        if taken is None:
            emitted.append(best if temperature <= 0 else draw(rest, float(u[0])))
            return emitted, path
        emitted.append(int(tokens[taken]))
        path.append(taken)
        node = taken


def commit(kv, table, base, path, block_size, scales=()):
    """One row: moves the kept nodes' rows of kv [2, layers, blocks, block, heads, dim] (and of each [layers, blocks,
    block] scale tensor) in place."""
    old, old_scales = kv.clone(), [s.clone() for s in scales]
    for place, node in enumerate(path):
        a, z = base + node, base + place
        kv[:, :, table[z // block_size], z % block_size] = old[:, :, table[a // block_size], a % block_size]
        for s, o in zip(scales, old_scales):
            s[:, table[z // block_size], z % block_size] = o[:, table[a // block_size], a % block_size]
