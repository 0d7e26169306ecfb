"""Speculative decoding over the paged cache: several drafted tokens of every sequence are checked in one
forward pass of the target model (src/inference/speculative.py, which runs HuggingFace models over chains and
bypasses the paged path).

A row drafts a tree of at most 256 nodes.  Node 0 is the last accepted token, whose K and V are not cached yet;
parents[i] < i is the node that node i follows; siblings are alternatives for the same place, in the order in which
they are to be tried.  A step:

    positions, slots, mask = draft_layout(parents, context_lens, block_tables, block_size, num_blocks)
    ... the model's layers over tokens [batch * nodes]: node i's K and V go to `slots`, then
        out = paged_draft_attention(q, k_cache, v_cache, block_tables, context_lens, mask, scale)
    tokens, counts, path = verify_drafts(logits, draft_tokens, uniforms, parents)
    context_lens = commit_drafts(kv_cache, block_tables, context_lens, path, counts)

ModelRunner.run_drafts() is the middle line for a model of PagedAttention layers.  context_lens counts the committed
tokens throughout; num_nodes (int32 [batch]) says how many nodes a row really drafts, 0 for a padded row.  Nothing
here synchronises with the host, so a step can be recorded in a HIP graph (after a warm-up run inside
attention.sizing_graph_workspace(), as for paged_decode; graphs that replay at the same time need workspaces of their own).
"""
import functools

import torch

from . import _native
from .attention import (_check_cache, _code, _compute_units, _debug_tables, _int32, _require_gpu, _stream_ptr,
                        check_block_tables, reserve_decode_workspace)

MAX_DRAFT_NODES = 256

_get_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


@functools.lru_cache(maxsize=1024)
def _attention_workspace(batch, nodes, num_q_heads, head_dim, parts):
    return _native.load().pa_draft_workspace_bytes(batch, nodes, num_q_heads, head_dim, parts)


@functools.lru_cache(maxsize=1024)
def _verify_workspace(batch, nodes, vocab):
    return _native.load().pa_verify_workspace_bytes(batch, nodes, vocab)


def _same_device(what, first, *others):
    """Launches go to the current device, whose index this returns: every tensor has to be there."""
    index = first.get_device()
    if index < 0:
        _require_gpu(first, what)
    for t in others:
        if t is not None and t.get_device() != index:
            raise RuntimeError("%s: tensors on %s and %s" % (what, first.device, t.device))
    if index != _get_device():
        raise RuntimeError("%s: the tensors are on %s, the current device is cuda:%d (use torch.cuda.device)"
                           % (what, first.device, _get_device()))
    return index


def _tables(block_tables, batch, what):
    """(int32 tensor, stride between rows, columns)"""
    shape = block_tables.shape
    if len(shape) != 2 or shape[0] != batch:
        raise RuntimeError("%s: block_tables must be [batch, max_blocks]" % what)
    if block_tables.dtype != torch.int32:
        block_tables = block_tables.to(torch.int32)
    row, column = block_tables.stride()
    if column != 1 or row < shape[1]:
        block_tables, row = block_tables.contiguous(), shape[1]
    return block_tables, row, shape[1]


def _lengths(t, batch, name, what):
    if t is None:
        return None
    if t.numel() != batch:
        raise RuntimeError("%s: %s must have one entry per row" % (what, name))
    return _int32(t, what)


def _trees(parents, batch, nodes, what):
    """(int32 tensor, stride between rows): stride 0 for one tree that every row drafts."""
    parents = _int32(parents, what)
    shape = parents.shape
    if len(shape) == 1 and shape[0] == nodes:
        return parents, 0
    if shape != (batch, nodes):
        raise RuntimeError("%s: parents must be [nodes] or [batch, nodes]" % what)
    return parents, nodes


def draft_layout(parents, context_lens, block_tables=None, block_size=16, num_blocks=None, num_nodes=None):
    """Where the drafted nodes of a step sit and which of them each one descends from:
    (positions int64 [batch, nodes], slots int32 [batch, nodes] or None, tree_mask int64 [batch or 1, nodes, words]).

    parents int32 [nodes] (one tree for every row) or [batch, nodes], parents[i] < i, -1 for node 0; context_lens
    int32 [batch], the committed tokens.  A node's position (for the rotary embedding) is context_len + its depth, its
    cache slot that of position context_len + its index; nodes past num_nodes get position 0 and slot -1, which the KV
    writers skip, as do nodes whose position lies outside the block table or the pool.  Bit j % 64 of word j / 64 of a
    mask row is set where node j is the node itself or one of its ancestors."""
    what = "draft_layout"
    device = _same_device(what, context_lens, parents, block_tables, num_nodes)
    lib = _native.load()
    lens = _int32(context_lens, what)
    batch = lens.numel()
    if parents.dim() not in (1, 2):
        raise RuntimeError("%s: parents must be [nodes] or [batch, nodes]" % what)
    nodes = parents.shape[-1]
    if not 1 <= nodes <= MAX_DRAFT_NODES:
        raise RuntimeError("%s: a row drafts 1 to %d nodes, got %d" % (what, MAX_DRAFT_NODES, nodes))
    parents, stride = _trees(parents, batch, nodes, what)
    real = _lengths(num_nodes, batch, "num_nodes", what)
    positions = lens.new_empty((batch, nodes), dtype=torch.int64)
    mask = positions.new_empty((batch if stride else 1, nodes, (nodes + 63) // 64))
    slots = tables = tables_ptr = slots_ptr = None
    row = width = 0
    if block_tables is not None:
        if num_blocks is None:
            raise RuntimeError("%s: num_blocks is needed with block_tables" % what)
        tables, row, width = _tables(block_tables, batch, what)
        slots = lens.new_empty((batch, nodes))
        tables_ptr, slots_ptr = tables.data_ptr(), slots.data_ptr()
    if batch == 0:
        return positions, slots, mask
    rc = lib.pa_draft_layout(parents.data_ptr(), stride, lens.data_ptr(), real.data_ptr() if real is not None else None,
                             tables_ptr, row, width, positions.data_ptr(), slots_ptr, mask.data_ptr(), batch, nodes,
                             int(block_size), 1 if num_blocks is None else int(num_blocks), _stream_ptr(device))
    _native.check(rc, "pa_draft_layout")
    return positions, slots, mask


# ---- how an attention launch is shaped -----------------------------------------------------------------------
# Rows (node, query head of a group) a workgroup serves from one pass over K and V -> workgroups a CU holds at once, what a
# token costs (ns) a workgroup that has its CU to itself and one that shares it, what a round of workgroups costs besides (ns),
# the bytes per ns that a launch of them draws from HBM.  A launch lasts as long as its rounds of workgroups and the memory
# need, neither quite hidden behind the other; a split adds the merge pass and the partial results it writes and reads.
# Fitted to a sweep of tiles and splits on an MI355X (19 shapes: batch 1 to 64, 5 to 64 nodes, 512 to 32k tokens, ratios of 2
# to 8, head_dim 128, fp16, bf16 and fp8 caches, K and V cold): the choice is 1 % above the sweep's best on average, 5 % at
# worst (profiles/drafted_attention_launch_sweep.txt).  head_dim enters by the bytes alone, though a token of 64 is staged and
# multiplied in less time: over 6 such shapes the choice is 3 % above the best on average, 11 % at worst.  Wide workgroups pay
# also where they are half empty, since they have the most loads in flight: 24 rows of 10 nodes x 4 query heads a KV head x
# 3000 tokens take 57 us with 128 rows a workgroup, 76 with 64, 93 with 32.
_DRAFT_TILES = {16: (2, 9.6, 9.1, 2700.0, 6800.0), 32: (2, 9.8, 8.4, 5600.0, 6300.0), 64: (2, 18.4, 11.6, 2900.0, 6700.0),
                128: (1, 16.7, 16.7, 4100.0, 9000.0)}
_DRAFT_LAUNCH_NS = 5400.0
_DRAFT_MERGE_NS = (3000.0, 1.0)      # the pass, per partition
_DRAFT_PARTIAL_BYTES_PER_NS = 2450.0
_DRAFT_MIN_PARTITION = 96            # tokens
_DRAFT_MAX_PARTITIONS = 64


@functools.lru_cache(maxsize=4096)
def _choose_draft_launch(batch, nodes, num_q_heads, num_kv_heads, head_dim, elem_bytes, max_keys, mean_keys, compute_units):
    """(rows per workgroup, partition_size, max_partitions) with the smallest modelled time; (.., 0, 1): one pass."""
    rows = nodes * (num_q_heads // num_kv_heads)
    read = batch * num_kv_heads * mean_keys * 2.0 * head_dim * elem_bytes
    # a batch of unequal rows: a row of the mean length counts its whole partitions and half a one at its end
    ragged = mean_keys < 0.9 * max_keys
    best = None
    for tile, (per_cu, alone, shared, round_ns, rate) in _DRAFT_TILES.items():
        if tile > 16 and 4 * rows <= tile:
            continue
        row_tiles = -(-rows // tile)
        memory = read / rate
        full = max(alone, per_cu * shared) if per_cu > 1 else alone
        for want in range(1, min(_DRAFT_MAX_PARTITIONS, -(-max_keys // _DRAFT_MIN_PARTITION)) + 1):
            size = -(-(-(-max_keys // want)) // 32) * 32
            parts = -(-max_keys // size)
            live = batch * (mean_keys / size + 0.5) if ragged and parts > 1 else batch * parts
            rounds, rest = divmod(-(-live * num_kv_heads * row_tiles // compute_units), per_cu)
            compute = min(size, max_keys) * (rounds * full + (alone if rest else 0.0)) + round_ns * (rounds + (1 if rest else 0))
            cost = _DRAFT_LAUNCH_NS + (memory * memory + compute * compute) ** 0.5
            if parts > 1:
                partials = live * nodes * num_q_heads * head_dim * 4.0
                cost += _DRAFT_MERGE_NS[0] + _DRAFT_MERGE_NS[1] * parts + 2.0 * partials / _DRAFT_PARTIAL_BYTES_PER_NS
            if best is None or cost < best[0]:
                best = (cost, tile, size, parts)
    _, tile, size, parts = best
    return (tile, size, parts) if parts > 1 else (tile, 0, 1)


def paged_draft_attention(q, k_cache, v_cache, block_tables, context_lens, tree_mask, scale, k_scale=None, v_scale=None,
                          num_nodes=None, out=None, partition_size=None, workspace=None, longest_context=None,
                          mean_context=None):
    """Attention of the drafted nodes q [batch, nodes, heads, head_dim] over the paged cache: node i attends to the row's
    context_lens committed tokens and to the nodes of its mask (draft_layout's tree_mask [batch or 1, nodes, words]), whose
    K and V have been written at cache positions context_len + node.  Returns [batch, nodes, heads, head_dim]; zeros for
    nodes past num_nodes and for a node that sees nothing.  Infinities and NaN in what a node sees, and in its query, come out as
    the formula has it.  Queries of another type than a 16-bit cache's, or over an fp8 one, are multiplied as fp16 (bf16
    exactly, fp32 to 11 bits, of any size), the K and V of a bf16 cache too then: beyond 65504 they count as infinite.

    A q of [batch * nodes, heads, head_dim] is taken too (and gives such an output); nodes then is the mask's.
    partition_size None: the launch policy's split of a row's tokens (the result does not depend on it beyond fp32
    rounding), 0: none, else a multiple of 32.  workspace: a uint8 tensor for the partitions' partial results instead of
    the device's shared one.  longest_context / mean_context: what the host knows about context_lens, as for paged_decode;
    wrong values cost time, never correctness."""
    what = "paged_draft_attention"
    device = _same_device(what, q, k_cache, v_cache, block_tables, context_lens, tree_mask, k_scale, v_scale, num_nodes, out,
                          workspace)
    _check_cache(k_cache, v_cache, what)
    lib = _native.load()
    batch = context_lens.numel()
    masks = tree_mask.shape
    if len(masks) != 3 or tree_mask.dtype != torch.int64 or masks[0] not in (1, batch):
        raise RuntimeError("%s: tree_mask must be int64 [batch or 1, nodes, words]" % what)
    nodes = masks[1]
    if not 1 <= nodes <= MAX_DRAFT_NODES or masks[2] != (nodes + 63) // 64:
        raise RuntimeError("%s: tree_mask %s is not one of 1 to %d nodes" % (what, tuple(masks), MAX_DRAFT_NODES))
    shape = q.shape
    if (shape[:2] != (batch, nodes)) if len(shape) == 4 else (len(shape) != 3 or shape[0] != batch * nodes):
        raise RuntimeError("%s: q %s does not match %d rows of %d nodes" % (what, tuple(shape), batch, nodes))
    num_q_heads, head_dim = shape[-2:]
    num_blocks, block_size, num_kv_heads, d2 = k_cache.shape
    if d2 != head_dim:
        raise RuntimeError("%s: q head_dim %d != cache head_dim %d" % (what, head_dim, d2))
    flat, q_stride, dense = q, num_q_heads * head_dim, q.is_contiguous()
    if not dense:
        flat = q if len(shape) == 3 else q.reshape(batch * nodes, num_q_heads, head_dim)
        if (flat.stride(2) != 1 or flat.stride(1) != head_dim or flat.stride(0) * flat.element_size() % 16
                or (flat.shape[0] > 1 and flat.stride(0) < q_stride)):
            flat = flat.contiguous()
        elif flat.shape[0] > 1:
            q_stride = flat.stride(0)
    if flat.data_ptr() % 16:
        flat, q_stride = flat.clone(memory_format=torch.contiguous_format), num_q_heads * head_dim
    tables, tables_row, width = _tables(block_tables, batch, what)
    lens = _int32(context_lens, what)
    real = _lengths(num_nodes, batch, "num_nodes", what)
    mask = tree_mask.contiguous()
    if out is None:
        out = torch.empty_like(q) if dense else torch.empty(shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous():
        raise RuntimeError("%s: out must be contiguous and like q" % what)
    if batch == 0:
        return out
    if width == 0:
        raise RuntimeError("%s: block_tables without columns" % what)
    kv_code = _code(k_cache.dtype, what)
    scales = (None, None)
    fp8 = kv_code == _native.DTYPE_FP8_E4M3
    if fp8:
        for t in (k_scale, v_scale):
            if t is None or t.dtype != torch.float32 or t.numel() != num_blocks * block_size or not t.is_contiguous():
                raise RuntimeError("%s: an fp8 cache needs contiguous fp32 k_scale and v_scale [num_blocks, block_size]" % what)
        scales = (k_scale.data_ptr(), v_scale.data_ptr())
    if _debug_tables():
        bad, short = check_block_tables(tables, lens + (real if real is not None else nodes), block_size, num_blocks)
        if bad or short:
            raise RuntimeError("%s: %d block-table entries outside the pool of %d blocks, %d rows whose tokens need more "
                               "than the table's %d columns" % (what, bad, num_blocks, short, width))
    if partition_size is None:
        bound = width * block_size
        if longest_context and longest_context > 0:
            bound = min(bound, -(-(int(longest_context) + nodes) // 256) * 256)
        # sixteenths of the bound: batches of about the same shape share the decision
        mean = bound if not mean_context else max(1, min(16, round(16.0 * (mean_context + nodes) / bound))) * bound // 16
        tile, psize, parts = _choose_draft_launch(batch, nodes, num_q_heads, max(1, num_kv_heads), head_dim, k_cache.element_size(),
                                                  bound, mean, _compute_units(q.device))
    else:
        tile, psize = 0, int(partition_size)
        parts = max(1, -(-width * block_size // psize)) if psize > 0 else 1
    ws_ptr, ws_bytes = None, 0
    if parts > 1:
        ws_bytes = _attention_workspace(batch, nodes, num_q_heads, head_dim, parts)
        if workspace is not None:
            if workspace.dtype != torch.uint8 or workspace.numel() < ws_bytes or not workspace.is_contiguous():
                raise RuntimeError("%s: workspace must be a contiguous uint8 GPU tensor of at least %d bytes" % (what, ws_bytes))
            ws = workspace
        else:
            ws = reserve_decode_workspace(q.device, ws_bytes)
        ws_ptr = ws.data_ptr()
    rc = lib.pa_draft_attention(flat.data_ptr(), _code(q.dtype, what), q_stride, k_cache.data_ptr(), v_cache.data_ptr(), *scales,
                                kv_code, tables.data_ptr(), tables_row, width, lens.data_ptr(),
                                real.data_ptr() if real is not None else None, mask.data_ptr(),
                                nodes * masks[2] if masks[0] > 1 else 0, out.data_ptr(), num_q_heads * head_dim, batch, nodes,
                                num_q_heads, num_kv_heads, head_dim, block_size, num_blocks, float(scale), psize, parts, ws_ptr,
                                ws_bytes, tile, _stream_ptr(device))
    _native.check(rc, "pa_draft_attention")
    return out


def verify_drafts(logits, draft_tokens, uniforms=None, parents=None, num_nodes=None, draft_probs=None, temperature=0.7,
                  top_p=0.9, generator=None, workspace=None):
    """Which drafted nodes the target accepts, and the token that follows them:
    (tokens int64 [batch, nodes], counts int32 [batch], path int32 [batch, nodes]).

    logits [batch, nodes, vocab] are the target's after every node (node 0: after the last accepted token), draft_tokens
    int64 [batch, nodes] the drafted ids (node 0's is not read).  parents as for draft_layout, None: a chain.
    tokens[b, :counts[b]] are what the row emits - the accepted tokens and the one after them - and path[b, :counts[b]] the
    nodes whose K and V stay, in ascending order, node 0 first; -1 beyond.  Rows of num_nodes 0 emit nothing.

    temperature and top_p select the target's distribution as in sample_tokens, temperature <= 0 is greedy.  Node c's
    token is accepted against uniforms[b, c], the token after the last accepted node is drawn with uniforms[b, 0]
    (fp32 [batch, nodes] in [0, 1); drawn here from `generator` by default).  draft_probs [batch, nodes - 1, vocab]: the
    distribution each chain token was drawn from, the row of its parent; without it the drafts are taken as
    certain and accepted with the target's probability, siblings one after the other with what the earlier ones leave.
    Either way the emitted tokens are distributed as the target's own samples."""
    what = "verify_drafts"
    index = _same_device(what, logits, draft_tokens, uniforms, parents, num_nodes, draft_probs, workspace)
    if logits.dim() != 3:
        raise RuntimeError("%s: logits must be [batch, nodes, vocab], got %s" % (what, tuple(logits.shape)))
    batch, nodes, vocab = logits.shape
    if not 1 <= nodes <= MAX_DRAFT_NODES:
        raise RuntimeError("%s: a row drafts 1 to %d nodes, got %d" % (what, MAX_DRAFT_NODES, nodes))
    if draft_tokens.shape != (batch, nodes) or draft_tokens.dtype != torch.int64:
        raise RuntimeError("%s: draft_tokens must be int64 [batch, nodes]" % what)
    lib = _native.load()
    temperature, top_p = float(temperature), float(top_p)
    device = logits.device
    if not logits.is_contiguous() and (logits.stride(2) != 1 or (nodes > 1 and logits.stride(1) < vocab)
                                       or (batch > 1 and logits.stride(0) < vocab)):
        logits = logits.contiguous()
    tokens = draft_tokens.contiguous()
    tokens_out = torch.empty_like(tokens)
    counts = torch.empty(batch, dtype=torch.int32, device=device)
    path = counts.new_empty((batch, nodes))
    if batch == 0:
        return tokens_out, counts, path
    stride = 0
    if parents is not None:
        parents, stride = _trees(parents, batch, nodes, what)
    real = _lengths(num_nodes, batch, "num_nodes", what)
    if temperature > 0:
        if uniforms is None:
            uniforms = torch.rand((batch, nodes), device=device, dtype=torch.float32, generator=generator)
        if uniforms.shape != (batch, nodes) or uniforms.dtype != torch.float32:
            raise RuntimeError("%s: uniforms must be fp32 [batch, nodes]" % what)
        uniforms = uniforms.contiguous()
    probs = None
    if draft_probs is not None:
        if parents is not None:
            raise RuntimeError("%s: draft_probs go with chains (parents=None) only" % what)
        if draft_probs.shape != (batch, nodes - 1, vocab):
            raise RuntimeError("%s: draft_probs must be [batch, nodes - 1, vocab], got %s" % (what, tuple(draft_probs.shape)))
        if nodes > 1 and temperature > 0:
            probs = draft_probs
            if probs.stride(2) != 1 or (nodes > 2 and probs.stride(1) < vocab) or (batch > 1 and probs.stride(0) < vocab):
                probs = probs.contiguous()
    ws_bytes = _verify_workspace(batch, nodes, vocab)
    if workspace is None:
        workspace = reserve_decode_workspace(device, ws_bytes)
    elif workspace.dtype != torch.uint8 or workspace.numel() < ws_bytes or not workspace.is_contiguous():
        raise RuntimeError("%s: workspace must be a contiguous uint8 GPU tensor of at least %d bytes" % (what, ws_bytes))
    rc = lib.pa_verify_drafts(logits.data_ptr(), _code(logits.dtype, what), logits.stride(1) if nodes > 1 else vocab,
                              logits.stride(0) if batch > 1 else 0, tokens.data_ptr(),
                              uniforms.data_ptr() if temperature > 0 else None,
                              parents.data_ptr() if parents is not None else None, stride,
                              real.data_ptr() if real is not None else None, probs.data_ptr() if probs is not None else None,
                              _code(probs.dtype, what) if probs is not None else 0,
                              (probs.stride(1) if nodes > 2 else vocab) if probs is not None else 0,
                              (probs.stride(0) if batch > 1 else 0) if probs is not None else 0, temperature, top_p,
                              batch, nodes, vocab, tokens_out.data_ptr(), counts.data_ptr(), path.data_ptr(),
                              workspace.data_ptr(), ws_bytes, _stream_ptr(index))
    _native.check(rc, "pa_verify_drafts")
    return tokens_out, counts, path


def commit_drafts(kv_cache, block_tables, context_lens, path, counts, k_scale=None, v_scale=None):
    """Move the kept nodes' K and V, in every layer, to consecutive cache positions; returns the new context_lens
    (int32 [batch], context_lens + counts).

    kv_cache [2, layers, num_blocks, block_size, kv_heads, head_dim], contiguous (BlockPool.kv_cache_tensor), changed in
    place; k_scale / v_scale [layers, num_blocks, block_size] of an fp8 pool, changed with it.  path and counts as
    verify_drafts returns them.  The blocks that hold the drafted positions must be the row's own (a shared last block
    is copied before it is written, as for any decode step); those behind the next token's are free again, and have to
    leave a row's table before ModelRunner.prepare_decode() sees it."""
    what = "commit_drafts"
    device = _same_device(what, kv_cache, block_tables, context_lens, path, counts, k_scale, v_scale)
    if kv_cache.dim() != 6 or kv_cache.shape[0] != 2 or not kv_cache.is_contiguous():
        raise RuntimeError("%s: kv_cache must be contiguous [2, layers, num_blocks, block_size, kv_heads, head_dim]" % what)
    lib = _native.load()
    _, layers, num_blocks, block_size, heads, head_dim = kv_cache.shape
    if layers == 0:      # the launch that moves the rows of the layers writes the lengths, too
        raise RuntimeError("%s: a pool without layers" % what)
    lens = _int32(context_lens, what)
    if lens.dim() != 1:
        lens = lens.view(-1)
    batch = lens.numel()
    if path.dim() != 2 or path.shape[0] != batch or path.shape[1] > MAX_DRAFT_NODES:
        raise RuntimeError("%s: path must be [batch, nodes] of at most %d nodes" % (what, MAX_DRAFT_NODES))
    path = _int32(path, what)
    counts = _lengths(counts, batch, "counts", what)
    tables, tables_row, width = _tables(block_tables, batch, what)
    es = kv_cache.element_size()
    fp8 = es == 1
    if fp8:
        for t in (k_scale, v_scale):
            if t is None or t.dtype != torch.float32 or t.numel() != layers * num_blocks * block_size or not t.is_contiguous():
                raise RuntimeError("%s: an fp8 pool needs contiguous fp32 k_scale and v_scale [layers, num_blocks, block_size]" % what)
    new_lens = torch.empty_like(lens)
    if batch == 0:
        return new_lens
    row = heads * head_dim * es
    rc = lib.pa_draft_commit(kv_cache.data_ptr(), layers, num_blocks * block_size * row, row,
                             k_scale.data_ptr() if fp8 else None, v_scale.data_ptr() if fp8 else None, num_blocks * block_size,
                             tables.data_ptr(), tables_row, width, lens.data_ptr(), path.data_ptr(), path.shape[1],
                             counts.data_ptr(), new_lens.data_ptr(), batch, path.shape[1], block_size, num_blocks,
                             _stream_ptr(device))
    _native.check(rc, "pa_draft_commit")
    return new_lens
