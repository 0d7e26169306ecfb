"""Speculative decoding on the GPU where values are no ordinary numbers or sizes no ordinary ones: NaN and infinities in
committed tokens and queries, at every width of a workgroup and split of a row, element by element against the 64-bit oracle."""
import math
import random

import pytest
import torch

from oracle import speculative_oracle as so
from test_gpu_drafts import DT, FP8, Pool, bound, check_verify, make_parents, one_width      # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def i32(values, gpu):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


def check_elements(pa, gpu, pool, q, lens, sets, partitions, p_type, scale=None, real=None):
    """Every output element against the oracle: where that is NaN or infinite the output is the same, elsewhere it is within
    bound().  q [batch, nodes, heads, dim] on the CPU."""
    batch, nodes, hq, dim = q.shape
    scale = dim ** -0.5 if scale is None else scale
    mask = torch.stack([so.mask_words(s, nodes) for s in sets]).to(gpu)
    k, v, tables, ks, vs = pool.device(gpu)
    outs = [pa.paged_draft_attention(q.to(gpu), k, v, tables, i32(lens, gpu), mask, scale, ks, vs, partition_size=part,
                                     num_nodes=None if real is None else i32(real, gpu)).cpu()
            for part in partitions]
    odd = 0
    for b in range(batch):
        n = nodes if real is None else real[b]
        kr, vr = (so.row_kv(x, f, pool.tables[b].tolist(), lens[b] + n, pool.block) for x, f in ((pool.k, pool.ks), (pool.v, pool.vs)))
        want, spread, weight = so.attention(q[b], kr, vr, lens[b], sets[b], n, scale)
        fine = torch.isfinite(want)
        odd += int((~fine).sum())
        for part, out in zip(partitions, outs):
            got = out[b].double()
            assert torch.equal(torch.isnan(got), torch.isnan(want)), (b, part)
            assert torch.equal(torch.where(torch.isinf(got), got, 0.0), torch.where(torch.isinf(want), want, 0.0)), (b, part)
            far, may = (got - want).abs()[fine], bound(want, spread, weight, p_type, q.dtype)[fine]
            assert (far <= may).all(), (b, part, float((far / may).max()))
    return odd


def poison(t, scales, tables, block, row, pos, head, dims, value):
    """Token `pos` of a row, one KV head and some dims: NaN or an infinity (fp8: NaN, which is all it has)."""
    at = (int(tables[row, pos // block]), pos % block, head)
    if t.dtype == FP8:
        t.view(torch.uint8)[at][dims] = 0x7F
    else:
        t[at][dims] = value


TYPES = [("fp16", "fp16"), ("bf16", "bf16"), ("fp8", "fp16"), ("fp16", "bf16"), ("fp8", "fp32")]


def product_type(cache, q_type):
    return torch.bfloat16 if cache == "bf16" and q_type == "bf16" else torch.float16


def random_case(seed, lens, nodes, hq, hkv, dim, block, cache, q_type):
    rng = random.Random(seed)
    pool = Pool(seed, lens, [nodes] * len(lens), hkv, dim, block, cache)
    sets = [so.ancestors(make_parents("tree", nodes, rng)) for _ in lens]
    q = torch.randn(len(lens), nodes, hq, dim, generator=torch.Generator().manual_seed(seed + 1)).to(torch.float16).to(DT[q_type])
    return pool, sets, q


# ---------------------------------------------------------------------------------------------- infinities and NaN

@pytest.mark.parametrize("cache,q_type", TYPES)
@pytest.mark.parametrize("nodes", [3, 21])
def test_nan_and_infinity_in_committed_values(pa, gpu, one_width, cache, q_type, nodes):
    """V of committed tokens anywhere in a split: in its middle, in the last 32 tokens of partitions of an odd multiple of 32,
    just before the drafted tokens."""
    lens = [330, 70, 200]
    pool, sets, q = random_case(3, lens, nodes, 4, 2, 64, 16, cache, q_type)
    inf, nan = float("inf"), float("nan")
    for row, pos, head, dims, value in ((0, 70, 0, slice(0, 3), nan), (0, 95, 0, slice(3, 6), inf), (0, 159, 1, slice(8, 9), -inf),
                                        (0, 130, 1, slice(8, 11), inf), (0, 329, 0, slice(12, 13), inf), (0, 4, 1, slice(63, 64), nan),
                                        (1, 31, 0, slice(5, 6), -inf), (1, 69, 1, slice(0, 64), nan)):
        poison(pool.v, pool.vs, pool.tables, 16, row, pos, head, dims, value)
    odd = check_elements(pa, gpu, pool, q, lens, sets, (0, 32, 64, 96, 160, None), product_type(cache, q_type))
    assert odd == nodes * 2 * (7 + 4 + 1 + 64)          # dims of the rows' KV heads, 2 query heads each


@pytest.mark.parametrize("cache,q_type", TYPES)
def test_nan_and_infinity_in_drafted_and_committed_values(pa, gpu, one_width, cache, q_type):
    lens, nodes = [90, 64, 0], 9
    pool, sets, q = random_case(5, lens, nodes, 4, 2, 64, 8, cache, q_type)
    for row, pos, head, dims, value in ((0, 80, 0, slice(0, 2), float("inf")), (0, 10, 0, slice(2, 3), float("inf")),
                                        (0, 92, 0, slice(1, 3), -float("inf")),
                                        (0, 94, 0, slice(4, 9), float("nan")), (1, 40, 1, slice(2, 3), float("nan")),
                                        (1, 66, 1, slice(20, 40), float("inf")), (2, 3, 0, slice(0, 8), -float("inf"))):
        poison(pool.v, pool.vs, pool.tables, 8, row, pos, head, dims, value)
    assert check_elements(pa, gpu, pool, q, lens, sets, (0, 32, 96, None), product_type(cache, q_type)) > 0


@pytest.mark.parametrize("cache,q_type", TYPES)
@pytest.mark.parametrize("nodes", [3, 21])
def test_a_query_with_nan_or_infinity_has_no_finite_output(pa, gpu, one_width, cache, q_type, nodes):
    """An overflow before the attention must not come out as a vector of zeros, whatever the width and the split; other
    nodes and heads are as they were."""
    lens = [130, 0, 65]
    pool, sets, q = random_case(7, lens, nodes, 4, 2, 64, 16, cache, q_type)
    q[0, 1, 2, 5] = float("nan")
    q[1, 0, 0, :] = float("nan")
    q[2, 2, 3, 63] = float("inf")
    q[2, 1, 0, 7] = -float("inf")
    assert check_elements(pa, gpu, pool, q, lens, sets, (0, 32, 96, None), product_type(cache, q_type)) == 4 * 64


@pytest.mark.parametrize("cache,q_type", TYPES)
def test_nan_and_infinity_in_keys(pa, gpu, one_width, cache, q_type):
    """A NaN key that is all a node sees of its partition, one among others, and (16-bit caches) infinite keys, whose score
    is an infinity of either sign."""
    lens, nodes = [64, 96, 33, 0], 4
    pool, _, q = random_case(9, lens, nodes, 4, 2, 64, 16, cache, q_type)
    sets = [so.ancestors([-1, 0, 0, 0]) for _ in lens]
    for row, pos, head, value in ((0, 64, 0, float("nan")), (0, 66, 1, float("nan")), (1, 10, 0, float("nan")),
                                  (2, 35, 1, float("inf")), (3, 2, 0, -float("inf"))):
        poison(pool.k, pool.ks, pool.tables, 16, row, pos, head, slice(3, 4), value)
    assert check_elements(pa, gpu, pool, q, lens, sets, (0, 32, 64, None), product_type(cache, q_type)) > 0


@pytest.mark.parametrize("part", [0, 32])
def test_scores_of_minus_infinity_alone_are_nan_and_no_key_is_zero(pa, gpu, one_width, part):
    """softmax of nothing but -inf is NaN; a node without any key is the documented zero."""
    pool, _, q = random_case(11, [0, 0, 40], 3, 2, 1, 64, 16, "fp16", "fp16")
    q[..., 0] = 1.0
    for row, pos in ((0, 0), (0, 1), (2, 41)):
        poison(pool.k, None, pool.tables, 16, row, pos, 0, slice(0, 1), -float("inf"))
    sets = [[{0}, {0, 1}, set()], [{0}, set(), {2}], [set(), {1}, set()]]
    odd = check_elements(pa, gpu, pool, q, [0, 0, 40], sets, (part,), torch.float16)
    assert odd == 2 * 2 * 64          # nodes 0 and 1 of row 0; row 2's node 1 has its committed tokens


# ---------------------------------------------------------------------------------------------- queries of another type

@pytest.mark.parametrize("cache,q_type", [("fp16", "bf16"), ("fp16", "fp32"), ("fp8", "bf16"), ("fp8", "fp32"), ("bf16", "fp32")])
@pytest.mark.parametrize("size", [2.0 ** 40, 2.0 ** 18, 2.0 ** -18, 2.0 ** -40])
def test_queries_beyond_the_range_of_fp16(pa, gpu, one_width, cache, q_type, size):
    """Queries of any size that their type holds, the scale taking it back; rows of several sizes side by side."""
    lens, nodes = [40, 0, 100], 11
    pool, sets, q = random_case(13, lens, nodes, 4, 2, 64, 16, cache, q_type)
    q *= size
    q[:, 3] *= 2.0 ** -9              # its scores all but vanish
    q[0, 2, 1] = 0.0
    q[:, 5, :, ::2] *= 2.0 ** -12     # small next to large
    check_elements(pa, gpu, pool, q, lens, sets, (0, 32), product_type(cache, q_type), scale=64 ** -0.5 / size)


# ---------------------------------------------------------------------------------------------- sizes

@pytest.mark.parametrize("dim", [64, 128])
def test_a_partition_longer_than_any_row(pa, gpu, lib, dim):
    """The C entry takes partition sizes up to 2^31 - 256: a row then has one partition, whatever its length."""
    lens, nodes, hq, hkv = [300, 5, 700], 6, 4, 2
    pool, sets, q = random_case(17, lens, nodes, hq, hkv, dim, 16, "fp16", "fp16")
    k, v, tables, _, _ = pool.device(gpu)
    mask = torch.stack([so.mask_words(s, nodes) for s in sets]).to(gpu)
    qd, lens_t = q.to(gpu), i32(lens, gpu)
    want = pa.paged_draft_attention(qd, k, v, tables, lens_t, mask, dim ** -0.5, partition_size=0)
    need = lib.pa_draft_workspace_bytes(3, nodes, hq, dim, 2)
    ws = torch.empty(need, dtype=torch.uint8, device=gpu)
    for size in (0x7fffff00, 1 << 30, 1024):
        out = torch.full_like(qd, 9.0)
        rc = lib.pa_draft_attention(qd.data_ptr(), 0, hq * dim, k.data_ptr(), v.data_ptr(), None, None, 0, tables.data_ptr(),
                                    tables.stride(0), tables.shape[1], lens_t.data_ptr(), None, mask.data_ptr(), mask[0].numel(),
                                    out.data_ptr(), hq * dim, 3, nodes, hq, hkv, dim, 16, pool.blocks, dim ** -0.5, size, 2,
                                    ws.data_ptr(), need, 0, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, lib.pa_last_error()
        # one partition in both: the merge multiplies and divides by its sum, then rounds the same value
        torch.testing.assert_close(out.float(), want.float(), rtol=2.0 ** -10, atol=2.0 ** -20)


@pytest.mark.parametrize("cache", ["fp16", "fp8"])
def test_commit_refuses_a_pool_without_layers(pa, gpu, cache):
    kv = torch.zeros(2, 0, 4, 8, 1, 64, device=gpu).to(DT[cache])
    lens, path = i32([3, 4], gpu), torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    scales = [torch.zeros(0, 4, 8, device=gpu)] * 2 if cache == "fp8" else []
    with pytest.raises(RuntimeError, match="layer"):
        pa.commit_drafts(kv, torch.zeros(2, 2, dtype=torch.int32, device=gpu), lens, path, i32([1, 1], gpu), *scales)


def test_layout_refuses_a_pool_without_blocks(pa, gpu):
    with pytest.raises(RuntimeError, match="pool"):
        pa.draft_layout(i32([-1, 0], gpu), i32([3], gpu), torch.zeros(1, 4, dtype=torch.int32, device=gpu), 16, 0)


def test_attention_refuses_a_table_without_columns_and_takes_any_hint(pa, gpu):
    pool, sets, q = random_case(19, [40, 3], 3, 4, 2, 64, 16, "fp16", "fp16")
    k, v, tables, _, _ = pool.device(gpu)
    mask = torch.stack([so.mask_words(s, 3) for s in sets]).to(gpu)
    call = lambda t, **kw: pa.paged_draft_attention(q.to(gpu), k, v, t, i32([40, 3], gpu), mask, 0.125, **kw)
    for part in (None, 0, 32):
        with pytest.raises(RuntimeError, match="block_tables"):
            call(tables[:, :0], partition_size=part)
    empty = pa.paged_draft_attention(q[:0].to(gpu), k, v, tables[:0, :0], i32([], gpu), mask[:1], 0.125)
    assert empty.shape == (0, 3, 4, 64)           # no rows, no table
    want = call(tables, partition_size=0)
    # two roundings of the probabilities (bound()'s 2^-11 + 2^-13 of the values' size each) and of the output
    far = 2 * (2.0 ** -11 + 2.0 ** -13) * float(pool.vf.abs().max())
    for longest, mean in ((-3, None), (-400, -7.0), (1, 1.0), (1 << 40, 1e12), (5, 1e9)):
        torch.testing.assert_close(call(tables, longest_context=longest, mean_context=mean).float(), want.float(),
                                   rtol=2.0 ** -10, atol=far)


# ---------------------------------------------------------------------------------------------- verification

@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_greedy_without_a_finite_logit_takes_the_first_token(pa, gpu, dtype):
    """NaN counts as -inf, so the first maximum of a row of both is its first entry."""
    def none(x):
        x[0] = -float("inf")
        x[0, :, :3] = float("nan")
        x[1] = float("nan")
        x[1, :, 40:] = -float("inf")
        x[2] = -float("inf")
        x[3, :, :100] = float("nan")
    check_verify(pa, gpu, 71, 5, 4, 200, dtype, 0.0, 1.0, change=none)


def test_row_sums_of_large_vocabularies_of_32_bit_logits(pa, gpu):
    """4 million entries of 2^-39.99 beside one of 1: they weigh 1.007 * 2^-18 together, and a token of weight 1 passes iff
    u < 1 / (1 + 1.007 * 2^-18).  Numbers on either side of that, about 2^-19 away."""
    vocab = 1 << 22
    logits = torch.full((2, 2, vocab), -39.99 * math.log(2.0), device=gpu)
    logits[:, :, 5] = 0.0
    u = torch.tensor([[0.0, 1 - 1.5 * 2.0 ** -18], [0.0, 1 - 0.5 * 2.0 ** -18]], device=gpu)
    tokens = torch.full((2, 2), 5, device=gpu)
    for top_p in (1 - 2.0 ** -20, 1.0):
        _, counts, _ = pa.verify_drafts(logits, tokens, u, temperature=1.0, top_p=top_p)
        assert counts.tolist() == [2, 1], top_p


# ---------------------------------------------------------------------------------------------- again and again

@pytest.mark.parametrize("cache,q_type", TYPES)
@pytest.mark.parametrize("part", [None, 0, 96])
def test_attention_gives_the_same_bits_every_time(pa, gpu, one_width, cache, q_type, part):
    lens, nodes = [500, 33, 0, 260], 19
    pool, sets, q = random_case(23, lens, nodes, 8, 2, 128, 16, cache, q_type)
    k, v, tables, ks, vs = pool.device(gpu)
    mask = torch.stack([so.mask_words(s, nodes) for s in sets]).to(gpu)
    call = lambda: pa.paged_draft_attention(q.to(gpu), k, v, tables, i32(lens, gpu), mask, 128 ** -0.5, ks, vs, partition_size=part)
    first = call()
    assert all(torch.equal(call(), first) for _ in range(10))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("top_p", [0.9, 1.0])
def test_verification_gives_the_same_tokens_every_time(pa, gpu, dtype, top_p):
    g = torch.Generator(device=gpu).manual_seed(29)
    logits = (torch.randn(16, 12, 20011, generator=g, device=gpu) * 2).to(DT[dtype])
    tokens = logits[:, 0].float().topk(12).indices
    u, par = torch.rand(16, 12, generator=g, device=gpu), i32([-1] + [0] * 7 + [1, 2, 3, 4], gpu)
    call = lambda: pa.verify_drafts(logits, tokens, u, par, temperature=0.9, top_p=top_p)
    first = call()
    for _ in range(10):
        assert all(torch.equal(x, y) for x, y in zip(call(), first))


# ---------------------------------------------------------------------------------------------- far apart

@pytest.mark.parametrize("cache,q_type", [("fp16", "fp16"), ("fp8", "bf16")])
@pytest.mark.parametrize("rows", [16, 128])
def test_attention_and_commit_in_a_pool_beyond_32_bit_offsets(pa, gpu, monkeypatch, cache, q_type, rows):
    """The tokens' blocks lie at both ends of a K and a V plane of 5 GiB (fp8: 4.5 GiB)."""
    from ai_infra_train_infer_amd import _native
    from test_gpu_drafts import OneWidth
    lib = OneWidth(_native.load(), rows)
    monkeypatch.setattr(_native, "load", lambda: lib)
    lens, nodes, hkv, dim, block = [70, 33], 6, 8, 128, 16
    pool, sets, q = random_case(31, lens, nodes, 16, hkv, dim, block, cache, q_type)
    each = block * hkv * dim * (1 if cache == "fp8" else 2)
    big = (5 << 30) // each if cache == "fp16" else (9 << 29) // each
    far = torch.tensor([b if i % 2 else big - pool.blocks + b for i, b in enumerate(range(pool.blocks))])
    kv = torch.empty(2, 1, big, block, hkv, dim, dtype=DT[cache], device=gpu)
    scales = [torch.ones(1, big, block, device=gpu) for _ in range(2)] if cache == "fp8" else [None, None]
    raw = kv.view(torch.uint8).view(2, big, each)
    for i, t in enumerate((pool.k, pool.v)):
        raw[i, far.to(gpu)] = t.view(torch.uint8).view(pool.blocks, each).to(gpu)
    if cache == "fp8":
        scales[0][0, far.to(gpu)], scales[1][0, far.to(gpu)] = pool.ks.to(gpu), pool.vs.to(gpu)
    tables = torch.where(pool.tables >= 0, far.int()[pool.tables.clamp(min=0).long()], -1).to(gpu)
    mask = torch.stack([so.mask_words(s, nodes) for s in sets]).to(gpu)
    k, v, near, ks, vs = pool.device(gpu)
    layer = [None if s is None else s[0] for s in scales]
    for part in (0, 32):
        got = pa.paged_draft_attention(q.to(gpu), kv[0, 0], kv[1, 0], tables, i32(lens, gpu), mask, dim ** -0.5, *layer, partition_size=part)
        want = pa.paged_draft_attention(q.to(gpu), k, v, near, i32(lens, gpu), mask, dim ** -0.5, ks, vs, partition_size=part)
        assert torch.equal(got, want)
    path, counts = i32([[0, 2, 5, -1, -1, -1], [0, 1, 3, 4, -1, -1]], gpu), i32([3, 4], gpu)
    small = torch.stack([k, v])[:, None].contiguous()
    small_scales = [s[None].clone() for s in (ks, vs)] if cache == "fp8" else [None, None]
    a = pa.commit_drafts(kv, tables, i32(lens, gpu), path, counts, *scales)
    b = pa.commit_drafts(small, near, i32(lens, gpu), path, counts, *small_scales)
    assert torch.equal(a, b)
    assert torch.equal(raw[:, far.to(gpu)], small.view(torch.uint8).view(2, pool.blocks, each))
    if cache == "fp8":
        for x, y in zip(scales, small_scales):
            assert torch.equal(x[0, far.to(gpu)].nan_to_num(7.0), y[0].nan_to_num(7.0))


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_verification_of_rows_beyond_32_bit_offsets(pa, gpu, dtype):
    """Logits and draft probabilities whose rows are 2^30 entries and whose sequences 2^32 bytes and more apart."""
    g = torch.Generator().manual_seed(37)
    vocab, nodes, batch = 1003, 3, 2
    near = (torch.randn(batch, nodes, vocab, generator=g) * 2).to(DT[dtype]).to(gpu)
    q_near = torch.softmax(near[:, :-1].float() + 0.5 * torch.randn(batch, nodes - 1, vocab, generator=g).to(gpu), -1)
    tokens = torch.cat([torch.zeros(batch, 1, dtype=torch.long), torch.multinomial(q_near.cpu().view(-1, vocab), 1, generator=g).view(batch, -1)], 1).to(gpu)
    u = torch.rand(batch, nodes, generator=g).to(gpu)
    row, seq = (1 << 30) + 1, 3 * (1 << 30) + 7
    flat = torch.empty(seq + 2 * row + vocab, dtype=DT[dtype], device=gpu)
    far = flat.as_strided(near.shape, (seq, row, 1))
    far.copy_(near)
    q_flat = torch.empty(seq + row + vocab, device=gpu)
    q_far = q_flat.as_strided(q_near.shape, (seq, row, 1))
    q_far.copy_(q_near)
    for kw_far, kw_near in ((dict(), dict()), (dict(draft_probs=q_far), dict(draft_probs=q_near))):
        for temperature, top_p in ((0.0, 1.0), (0.9, 0.9), (1.0, 1.0)):
            a = pa.verify_drafts(far, tokens, u, temperature=temperature, top_p=top_p, **kw_far)
            b = pa.verify_drafts(near, tokens, u, temperature=temperature, top_p=top_p, **kw_near)
            assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 50.0, 1e6])
@pytest.mark.parametrize("top_p", [1.0, 0.9, 0.5])
def test_verify_at_extreme_temperatures(pa, gpu, dtype, temperature, top_p):
    """From one token that takes everything to weights that differ in the seventh digit."""
    check_verify(pa, gpu, 41, 6, 7, 331, dtype, temperature, top_p)
    check_verify(pa, gpu, 42, 4, 4, 17003, dtype, temperature, top_p, kind="chain", probs="fp32")
