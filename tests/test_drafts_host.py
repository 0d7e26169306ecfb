"""Speculative decoding without a GPU: the oracle against its definitions, the refusals of the wrappers and of the C
entry points (which check before they launch), the attention launch policy."""
import itertools

import pytest
import torch

from oracle import speculative_oracle as so


def test_ancestors_of_a_tree_a_chain_and_of_malformed_parents():
    assert so.ancestors([-1, 0, 0, 1, 1, 2]) == [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {0, 1, 4}, {0, 2, 5}]
    assert so.ancestors([-1, 0, 1, 2]) == [{0}, {0, 1}, {0, 1, 2}, {0, 1, 2, 3}]
    assert so.ancestors([5, 7, 1]) == [{0}, {1}, {1, 2}]
    assert so.mask_words([{0}, {0, 63}, {64}], 65).tolist()[:3] == [[1, 0], [1 - (1 << 63), 0], [0, 1]]


def _exhaust(logits, tokens_of, parents, probs, steps, first):
    """Distribution of the first `first` emitted tokens over all grids of uniform numbers (midpoints)."""
    n = len(parents)
    seen = {}
    grid = [(i + 0.5) / steps for i in range(steps)]
    for weight, tokens in tokens_of:
        for u in itertools.product(grid, repeat=n):
            out, _ = so.verify(logits, tokens, u, parents, n, 1.0, 1.0, probs)
            seen[tuple(out[:first])] = seen.get(tuple(out[:first]), 0.0) + weight / steps ** n
    return seen


@pytest.mark.parametrize("case", ["tree", "repeated sibling", "chain with probabilities"])
def test_emitted_tokens_have_the_targets_distribution(case):
    """The grid of midpoints is a quadrature in `steps` points per uniform number: an indicator of intervals is off
    by at most 1 / steps per comparison, and a token passes at most n of them."""
    logits = torch.log(torch.tensor([[0.5, 0.2, 0.3], [0.1, 0.6, 0.3], [0.25, 0.25, 0.5]], dtype=torch.float64))
    p = torch.softmax(logits, -1)
    steps = 24
    if case == "tree":
        got = _exhaust(logits, [(1.0, [0, 1, 0])], [-1, 0, 0], None, steps, 1)
    elif case == "repeated sibling":
        got = _exhaust(logits, [(1.0, [0, 2, 2])], [-1, 0, 0], None, steps, 1)
    else:
        q = torch.tensor([[0.2, 0.5, 0.3], [0.3, 0.3, 0.4]], dtype=torch.float64)
        # every pair of drafted tokens, weighted with the probability that the draft draws it
        pairs = [(float(q[0, a] * q[1, b]), [0, a, b]) for a in range(3) for b in range(3)]
        got = _exhaust(logits, pairs, [-1, 0, 1], q, 12, 1)
        steps = 12
    for t in range(3):
        assert abs(got.get((t,), 0.0) - float(p[0, t])) <= 3 / steps, (case, t, got)
    assert abs(sum(got.values()) - 1) < 1e-9


def test_greedy_chain_is_the_longest_matching_prefix():
    logits = torch.eye(4)[[2, 1, 3, 0]]
    for tokens, want in (([9, 2, 1, 3], ([2, 1, 3, 0], [0, 1, 2, 3])), ([9, 2, 0, 3], ([2, 1], [0, 1])), ([9, 0, 1, 3], ([2], [0]))):
        assert so.verify(logits, tokens, [0.0] * 4, [-1, 0, 1, 2], 4, 0.0, 1.0) == want


def test_nucleus_of_the_oracle():
    l = torch.log(torch.tensor([0.5, 0.3, 0.15, 0.05], dtype=torch.float64))
    kept = lambda p: (so.weights(l, 1.0, p) > 0).sum().item()
    assert [kept(x) for x in (0.4, 0.51, 0.79, 0.81, 0.94, 0.96, 1.0)] == [1, 2, 2, 3, 3, 4, 4]
    assert (so.weights(torch.tensor([1.0, 1.0, 0.0, float("nan"), -float("inf")]), 1.0, 0.1) > 0).tolist() == [True, True, False, False, False]


# ---------------------------------------------------------------------------------------------- refusals

def test_wrappers_refuse_cpu_tensors(pa):
    with pytest.raises(RuntimeError, match="GPU only"):
        pa.draft_layout(torch.tensor([-1, 0], dtype=torch.int32), torch.tensor([3], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="GPU only"):
        pa.verify_drafts(torch.zeros(1, 2, 8), torch.zeros(1, 2, dtype=torch.long))
    with pytest.raises(RuntimeError, match="GPU only"):
        pa.commit_drafts(torch.zeros(2, 1, 2, 8, 1, 64), None, None, None, None)
    with pytest.raises(RuntimeError, match="GPU only"):
        pa.paged_draft_attention(torch.zeros(1, 2, 2, 64), None, None, None, None, None, 1.0)


P = 4096        # an address that no refused call reads


def test_layout_c_abi_refusals(lib):
    good = dict(parents=P, stride=5, lens=P, real=None, tables=P, bt_stride=8, width=8, positions=P, slots=P, mask=P, batch=2,
                nodes=5, block=16, blocks=100, stream=None)
    call = lambda **kw: lib.pa_draft_layout(*{**good, **kw}.values())
    assert call(batch=0) == 0 and call(nodes=0) == 0
    for bad in (dict(parents=None), dict(lens=None), dict(positions=None), dict(mask=None), dict(batch=-1), dict(nodes=-1),
                dict(stride=4), dict(slots=None), dict(block=0), dict(blocks=0), dict(width=0), dict(bt_stride=7)):
        assert call(**bad) == -1, bad
        assert b"pa_draft_layout" in lib.pa_last_error()
    assert call(nodes=257, stride=257) == -2 and call(blocks=1 << 28) == -2


def test_fast_bindings_pass_doubles_and_floats(lib):
    """pa_verify_drafts takes two doubles, pa_draft_attention one float: the quick binding and ctypes agree on what the entry
    sees, tested through refusals that depend on the value."""
    need = lib.pa_verify_workspace_bytes(2, 5, 1000)
    for temperature, top_p, want in ((1e-7, 0.5, -2), (1.0, 0.0, -1), (0.5, -1.0, -1), (1e7, 0.5, -2), (float("nan"), 0.5, -1), (1, 0, -1)):
        args = (P, 0, 1000, 5000, P, P, None, 0, None, None, 2, 1000, 4000, temperature, top_p, 2, 5, 1000, P, P, P, P, need, None)
        assert lib.pa_verify_drafts(*args) == lib._cdll.pa_verify_drafts(*args) == want, (temperature, top_p)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        args = (P, 0, 2048, P, P, None, None, 0, P, 8, 8, P, None, P, 5, P, 2048, 2, 5, 16, 8, 128, 16, 100, scale, 64, 1, None, 0, 0, None)
        assert lib.pa_draft_attention(*args) == lib._cdll.pa_draft_attention(*args) == -1


def test_verify_c_abi_refusals(lib):
    need = lib.pa_verify_workspace_bytes(2, 5, 1000)
    assert need > 0 and lib.pa_verify_workspace_bytes(0, 5, 10) == 0
    good = dict(logits=P, dtype=0, row=1000, batch_stride=5000, tokens=P, uniforms=P, parents=None, pstride=0, real=None,
                probs=None, pdtype=2, prow=1000, pbatch=4000, temperature=1.0, top_p=0.9, batch=2, nodes=5, vocab=1000, out=P,
                counts=P, path=P, ws=P, ws_bytes=need, stream=None)
    call = lambda **kw: lib.pa_verify_drafts(*{**good, **kw}.values())
    assert call(batch=0) == 0
    for bad in (dict(logits=None), dict(tokens=None), dict(uniforms=None), dict(out=None), dict(counts=None), dict(path=None),
                dict(batch=-1), dict(nodes=0), dict(vocab=0), dict(row=999), dict(top_p=0.0), dict(top_p=float("nan")),
                dict(temperature=float("nan")), dict(parents=P, pstride=4), dict(probs=P, prow=999), dict(ws=P + 8)):
        assert call(**bad) == -1, bad
        assert b"pa_verify_drafts" in lib.pa_last_error()
    for bad in (dict(nodes=257), dict(batch=65536), dict(vocab=(1 << 24) + 1, row=1 << 25), dict(temperature=1e-7),
                dict(temperature=float("inf")), dict(parents=P, probs=P), dict(probs=P, pdtype=3), dict(dtype=3)):
        assert call(**{**bad, "ws_bytes": 1 << 40}) == -2, bad
    assert call(ws=None) == -4 and call(ws_bytes=need - 1) == -4


def test_commit_c_abi_refusals(lib):
    good = dict(pool=P, layers=2, plane=100 * 16 * 256, row=256, ks=None, vs=None, sstride=1600, tables=P, bt_stride=8, width=8,
                lens=P, path=P, pstride=5, counts=P, new=2 * P, batch=2, nodes=5, block=16, blocks=100, stream=None)
    call = lambda **kw: lib.pa_draft_commit(*{**good, **kw}.values())
    assert call(batch=0) == 0 and call(layers=0) == 0
    for bad in (dict(pool=None), dict(tables=None), dict(lens=None), dict(path=None), dict(counts=None), dict(new=None),
                dict(new=P), dict(ks=P), dict(batch=-1), dict(row=0), dict(bt_stride=7), dict(pstride=4), dict(block=0),
                dict(plane=100 * 16 * 256 - 16), dict(ks=P, vs=P, sstride=1599)):
        assert call(**bad) == -1, bad
        assert b"pa_draft_commit" in lib.pa_last_error()
    for bad in (dict(row=264, plane=100 * 16 * 264), dict(pool=P + 8), dict(nodes=257, pstride=257), dict(batch=65536),
                dict(blocks=1 << 28, plane=1 << 60)):
        assert call(**bad) == -2, bad


def test_attention_c_abi_refusals(lib):
    assert lib.pa_draft_workspace_bytes(2, 5, 16, 128, 1) == 0
    need = lib.pa_draft_workspace_bytes(2, 5, 16, 128, 4)
    assert need >= 2 * 5 * 16 * 4 * (128 + 2) * 4
    good = dict(q=P, qd=0, qs=2048, k=P, v=P, ks=None, vs=None, kd=0, tables=P, bt_stride=8, width=8, lens=P, real=None, mask=P,
                mstride=5, out=P, os=2048, batch=2, nodes=5, hq=16, hkv=8, dim=128, block=16, blocks=100, scale=0.1, psize=64,
                parts=4, ws=P, ws_bytes=need, tiles=0, stream=None)
    call = lambda **kw: lib.pa_draft_attention(*{**good, **kw}.values())
    assert call(batch=0) == 0 and call(nodes=0) == 0
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(tables=None), dict(lens=None), dict(mask=None), dict(out=None),
                dict(batch=-1), dict(hq=12), dict(hkv=0), dict(qs=2047), dict(os=2000), dict(q=P + 8), dict(mstride=4),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(tiles=4), dict(parts=0),
                dict(kd=3), dict(kd=3, ks=P, vs=P + 4), dict(width=0), dict(bt_stride=7), dict(blocks=0), dict(ws=P + 8)):
        assert call(**bad) == -1, bad
        assert b"pa_draft_attention" in lib.pa_last_error()
    for bad in (dict(nodes=257), dict(dim=96), dict(block=12), dict(block=4), dict(qd=3), dict(kd=2), dict(psize=48), dict(psize=0),
                dict(batch=65536), dict(hq=65536, hkv=8, qs=1 << 30, os=1 << 30)):
        assert call(**{**bad, "ws_bytes": 1 << 50}) == -2, bad
    assert call(ws=None) == -4 and call(ws_bytes=need - 1) == -4


def test_attention_launch_policy(pa):
    from ai_infra_train_infer_amd.speculative import _choose_draft_launch as choose
    for batch in (1, 3, 64, 400):
        for nodes in (1, 5, 33, 256):
            for heads, kv_heads in ((1, 1), (16, 8), (24, 3), (64, 8)):
                for keys in (1, 16, 127, 1000, 40000, 1 << 20):
                    for mean in {max(1, keys // 16), keys}:
                        tile, size, parts = choose(batch, nodes, heads, kv_heads, 128, 2, keys, mean, 256)
                        assert tile in (16, 32, 64, 128) and 1 <= parts <= 64
                        if parts == 1:
                            assert size == 0
                        else:       # the partitions cover every key, the last one at least one of them
                            assert size % 32 == 0 and (parts - 1) * size < keys <= parts * size
    # a lone sequence of 32k tokens is split over the chip, a batch that fills it is not
    assert choose(1, 5, 16, 8, 128, 2, 32768, 32768, 256)[2] > 8
    assert choose(256, 5, 16, 8, 128, 2, 512, 512, 256)[2] == 1
    # narrow tiles for chains, wide ones where many rows share the keys
    assert choose(1, 5, 16, 8, 128, 2, 4096, 4096, 256)[0] == 16
    assert choose(32, 64, 16, 8, 128, 2, 4096, 4096, 256)[0] == 128


def test_run_drafts_refuses_a_runner_without_a_model(pa):
    runner = pa.ModelRunner(None, pa.ModelRunnerConfig(block_size=16, device="cpu"))
    with pytest.raises(RuntimeError, match="tokens"):
        pa.ModelRunner(torch.nn.Identity(), runner.config).run_drafts(torch.zeros(2, 3).long(), torch.zeros(4).int(), torch.zeros(2, 1).int(), torch.zeros(2).int())
    one = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no model"):
        runner.run_drafts(one.long(), one, one, one[0])


@pytest.mark.parametrize("shared", [False, True])
def test_run_drafts_asks_the_model_for_no_id_behind_a_rows_nodes(pa, monkeypatch, shared):
    """verify_drafts pads its tokens with -1, and a padded row's ids can be anything: nodes without a slot must not reach the
    embedding, which reads its table at whatever id it gets."""
    from ai_infra_train_infer_amd import speculative

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.embed = torch.nn.Embedding(10, 4)

        def forward(self, ids, positions):
            self.ids = ids
            return self.embed(ids)

    def layout(parents, context_lens, tables, block_size, num_blocks, num_nodes):
        pos, slots = zip(*[so.layout(parents.tolist() if parents.dim() == 1 else parents[b].tolist(), int(context_lens[b]),
                                     int(num_nodes[b]) if context_lens[b] >= 0 else 0, tables[b].tolist(), block_size, num_blocks)[:2]
                           for b in range(len(context_lens))])
        return torch.tensor(pos), torch.tensor(slots, dtype=torch.int32), torch.zeros(1, 3, 1, dtype=torch.int64)

    monkeypatch.setattr(speculative, "draft_layout", layout)
    model = Model()
    runner = pa.ModelRunner(model, pa.ModelRunnerConfig(block_size=16, device="cpu"))
    tokens = torch.tensor([[3, -1, 5, 10], [9, 1 << 40, 6, 4], [-1, -7, 7, 4]]).t()       # in any order in memory
    kept = tokens.clone()
    parents = torch.tensor([-1, 0, 0], dtype=torch.int32)
    logits = runner.run_drafts(tokens, parents if shared else parents.expand(4, 3).contiguous(), torch.zeros(4, 2, dtype=torch.int32),
                               torch.tensor([4, 4, 4, -1], dtype=torch.int32), num_nodes=torch.tensor([2, 0, 3, 3], dtype=torch.int32))
    assert logits.shape == (4, 3, 4) and torch.equal(tokens, kept)
    assert model.ids.tolist() == [3, 9, 0, 0, 0, 0, 5, 6, 7, 0, 0, 0]
