"""A speculative step as it is used: layout, the model's forward over the drafts, verification and commit, one after the
other - eager, recorded in a HIP graph, on two streams at once - on the small Qwen3-shaped model of the other tests."""
import copy
import random

import pytest
import torch

from oracle import speculative_oracle as so
from test_gpu_drafts import Pool, make_parents
from test_gpu_model import Session, dense_reference_logits, small_model

pytestmark = pytest.mark.gpu


def i32(values, gpu):
    return torch.tensor(values, dtype=torch.int32, device=gpu)


class Speculating(Session):
    """A session whose rows hold token_ids; all but the last token of a row are in the cache (node 0 is the last one)."""

    def start(self, prompts):
        for p in prompts:
            self.add(p[:-1])
        self.prefill()
        for s, p in zip(self.seqs, prompts):
            s["token_ids"].append(p[-1])

    def tables(self, nodes, gpu):
        for s in self.seqs:
            self._grow(s, len(s["token_ids"]) - 1 + nodes)
        width = max(len(s["block_table"]) for s in self.seqs)
        return i32([s["block_table"] + [-1] * (width - len(s["block_table"])) for s in self.seqs], gpu)

    def lens(self):
        return [len(s["token_ids"]) - 1 for s in self.seqs]


def drafted(model, seqs, parents, nodes, vocab, rng):
    """Draft ids of which some branch is right: at every place one child (not always the first) carries the dense
    reference's greedy token while the path to it is right, the others other tokens."""
    rows = []
    for s, par in zip(seqs, parents):
        ids = [s["token_ids"][-1]] + [rng.randrange(vocab) for _ in range(nodes - 1)]
        text, node = list(s["token_ids"]), 0
        while True:
            children = [c for c in range(1, nodes) if par[c] == node]
            if not children or rng.random() < 0.2:
                break
            best = int(dense_reference_logits(model, text).argmax())
            node = rng.choice(children)
            ids[node] = best
            text.append(best)
        rows.append(ids)
    return rows


TOL = {"fp16": 3e-2, "fp8": 6e-2}     # what the decode tests of the same model allow its logits


@pytest.mark.parametrize("cache_dtype,psize,fused", [("fp16", 0, True), ("fp16", 32, False), ("fp8", 0, True)])
def test_steps_follow_the_dense_model(pa, gpu, cache_dtype, psize, fused):
    """Greedy steps over random trees: the logits of every node on the accepted path are the dense model's for the text
    that leads to it, the accepted tokens are its choices, and the next step, over the committed rows, still is."""
    rng = random.Random(7)
    model = small_model(pa, cache_dtype, psize, fused_qk=fused)
    ref = copy.deepcopy(model).half().float()
    sess = Speculating(pa, model, gpu, num_blocks=96, cache_dtype=cache_dtype)
    sess.start([[rng.randrange(512) for _ in range(n)] for n in (2, 17, 40, 65)])
    tol = TOL[cache_dtype]
    accepted = 0
    for nodes in (5, 1, 13, 20, 7):
        parents = [make_parents(rng.choice(["chain", "tree", "deep"]), nodes, rng) for _ in sess.seqs]
        ids = drafted(ref, sess.seqs, parents, nodes, 512, rng)
        tables, lens = sess.tables(nodes, gpu), sess.lens()
        par, toks, ctx = i32(parents, gpu), torch.tensor(ids, device=gpu), i32(lens, gpu)
        hints = {"longest_context": max(lens), "mean_context": sum(lens) / len(lens)} if nodes % 2 else {}
        logits = sess.runner.run_drafts(toks, par, tables, ctx, **hints)
        assert logits.shape == (4, nodes, 512) and pa.get_context().tree_mask is None
        out, counts, path = pa.verify_drafts(logits, toks, parents=par, temperature=0.0)
        after = sess.pool.commit_drafts(tables, ctx, path, counts).tolist()
        out, counts, path = out.tolist(), counts.tolist(), path.tolist()
        for b, s in enumerate(sess.seqs):
            assert counts[b] >= 1 and after[b] == lens[b] + counts[b]
            assert path[b][0] == 0 and all(c == -1 for c in path[b][counts[b]:])
            for j in range(counts[b]):
                want = dense_reference_logits(ref, s["token_ids"])
                torch.testing.assert_close(logits[b, path[b][j]].float().cpu(), want, rtol=tol, atol=tol)
                # the greatest of logits that are off by tol + tol |x| each
                assert want[out[b][j]] >= want.max() - 2 * tol * (1 + want.abs().max())
                if j + 1 < counts[b]:
                    assert parents[b][path[b][j + 1]] == path[b][j] and ids[b][path[b][j + 1]] == out[b][j]
                s["token_ids"].append(out[b][j])
            accepted += counts[b] - 1
    assert accepted >= 8        # the drafts hold the dense model's choices: paths of several nodes were committed
    for s in sess.seqs:         # the committed cache carries an ordinary decode step too
        s["done"] = len(s["token_ids"])
        sess._grow(s, s["done"])
        need = -(-s["done"] // 16)      # prepare_decode takes a table's last block as the last token's: the others go back
        sess.free += s["block_table"][need:]
        del s["block_table"][need:]
    got = sess.runner.run(*sess.runner.prepare_decode(sess.seqs), is_prefill=False)
    for b, s in enumerate(sess.seqs):
        torch.testing.assert_close(got[b].float().cpu(), dense_reference_logits(ref, s["token_ids"]), rtol=tol, atol=tol)


def test_padded_rows_and_short_trees_of_a_step(pa, gpu):
    """A row of num_nodes 0 writes nothing and emits nothing; a row that drafts fewer nodes is as if drafted alone."""
    rng = random.Random(3)
    model = small_model(pa)
    sess = Speculating(pa, model, gpu)
    sess.start([[rng.randrange(512) for _ in range(n)] for n in (30, 9, 50)])
    nodes, real = 9, [9, 0, 4]
    parents = [make_parents("tree", nodes, rng) for _ in real]
    tables, ctx = sess.tables(nodes, gpu), i32(sess.lens(), gpu)
    toks = torch.tensor([[rng.randrange(512) for _ in range(nodes)] for _ in real], device=gpu)
    par, num = i32(parents, gpu), i32(real, gpu)
    cache = sess.pool.kv_cache_tensor
    before = cache.clone()
    logits = sess.runner.run_drafts(toks, par, tables, ctx, num_nodes=num)
    out, counts, path = pa.verify_drafts(logits, toks, parents=par, num_nodes=num, temperature=0.0)
    after = sess.pool.commit_drafts(tables, ctx, path, counts)
    assert counts[1] == 0 and after[1] == ctx[1] and path[1].eq(-1).all() and out[1].eq(-1).all()
    touched = (cache != before).flatten(4).any(4).any(0).any(0)        # [blocks, block_size]
    allowed = torch.zeros_like(touched)
    for b in (0, 2):
        for i in range(real[b]):
            p = int(ctx[b]) + i
            allowed[tables[b, p // 16], p % 16] = True
    assert not (touched & ~allowed).any()
    cache.copy_(before)
    alone = sess.runner.run_drafts(toks[2:, :4], par[2:, :4].contiguous(), tables[2:], ctx[2:])
    # the same sums in another order and split: two logits that each are off by what the model tests allow
    torch.testing.assert_close(logits[2, :4].float(), alone[0].float(), rtol=6e-2, atol=6e-2)


def test_a_runner_without_a_model_refuses(pa, gpu):
    runner = pa.ModelRunner(None, pa.ModelRunnerConfig(block_size=16, device="cuda:0"))
    with pytest.raises(RuntimeError, match="no model"):
        runner.run_drafts(torch.zeros(1, 2, dtype=torch.int64, device=gpu), i32([-1, 0], gpu), i32([[0]], gpu), i32([3], gpu))


@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_a_captured_step_replays(pa, gpu, temperature):
    """The whole step as one graph, replayed with other inputs, eager steps and synchronisations between: each replay's
    verification is that of its own logits, its cache and lengths are those of the same step run eagerly."""
    from ai_infra_train_infer_amd.attention import sizing_graph_workspace
    rng = random.Random(11)
    model = small_model(pa)
    sess = Speculating(pa, model, gpu)
    sess.start([[rng.randrange(512) for _ in range(n)] for n in (30, 9, 50, 3)])
    nodes = 12
    tables, ctx = sess.tables(nodes + 60, gpu), i32(sess.lens(), gpu)
    toks = torch.zeros(4, nodes, dtype=torch.int64, device=gpu)
    par = i32([make_parents("tree", nodes, rng) for _ in range(4)], gpu)
    num, uni = i32([nodes] * 4, gpu), torch.rand(4, nodes, device=gpu)
    cache = sess.pool.kv_cache_tensor

    def step():
        logits = sess.runner.run_drafts(toks, par, tables, ctx, num_nodes=num)
        out = pa.verify_drafts(logits, toks, uni, par, num, temperature=temperature, top_p=0.9)
        return (logits, *out, sess.pool.commit_drafts(tables, ctx, out[2], out[1]))

    start = cache.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), sizing_graph_workspace():
        step()
    torch.cuda.current_stream().wait_stream(side)
    cache.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for replay in range(5):
        torch.cuda.synchronize()
        toks.copy_(torch.tensor([[rng.randrange(512) for _ in range(nodes)] for _ in range(4)]))
        par.copy_(torch.tensor([make_parents(rng.choice(["tree", "deep", "chain"]), nodes, rng) for _ in range(4)]))
        num.copy_(torch.tensor([nodes, rng.randrange(nodes + 1), 1, nodes]))
        uni.copy_(torch.rand(4, nodes, generator=torch.Generator().manual_seed(replay)))
        first = sess.runner.run_drafts(toks, par, tables, ctx, num_nodes=num).float()
        toks[:, 1:5] = first[:, 0].topk(4).indices        # likely tokens, so that something is accepted
        start = cache.clone()
        eager = [t.clone() for t in step()]
        eager_cache = cache.clone()
        cache.copy_(start)
        for _ in range(2):                                 # twice the same
            cache.copy_(start)
            graph.replay()
            torch.cuda.synchronize()
            logits, out, counts, path, after = (t.clone() for t in held)
            for b in range(4):
                n = int(num[b])
                torch.testing.assert_close(logits[b, :n].float(), eager[0][b, :n].float(), rtol=6e-2, atol=6e-2)
            again = pa.verify_drafts(logits, toks, uni, par, num, temperature=temperature, top_p=0.9)
            assert torch.equal(again[0], out) and torch.equal(again[1], counts) and torch.equal(again[2], path)
            assert torch.equal(after, ctx + counts)
            if torch.equal(logits, eager[0]):
                assert torch.equal(cache, eager_cache) and torch.equal(out, eager[1])
        ctx.copy_(after)


def test_two_graphs_with_their_own_workspaces_replay_together(pa, gpu):
    """Attention and verification of two graphs on two streams at once, each with a workspace of its own."""
    rng = random.Random(5)
    jobs = []
    for seed, nodes, vocab in ((1, 8, 9001), (2, 24, 7003)):
        lens = [700, 1300, 40]
        pool = Pool(seed, lens, [nodes] * 3, 2, 64, 16, "fp16")
        g = torch.Generator().manual_seed(seed)
        parents = make_parents("tree", nodes, rng)
        mask = so.mask_words(so.ancestors(parents), nodes)[None].to(gpu)
        jobs.append(dict(
            q=torch.randn(3, nodes, 8, 64, generator=g).half().to(gpu), kv=pool.device(gpu), lens=i32(lens, gpu), mask=mask,
            par=i32(parents, gpu), toks=torch.randint(0, 20, (3, nodes), generator=g).to(gpu),
            logits=(torch.randn(3, nodes, vocab, generator=g) * 3).half().to(gpu),
            uni=torch.rand(3, nodes, generator=g).to(gpu), ws=torch.empty(64 << 20, dtype=torch.uint8, device=gpu)))

    def run(j, own):
        ws = j["ws"] if own else None
        k, v, tables, _, _ = j["kv"]
        a = pa.paged_draft_attention(j["q"], k, v, tables, j["lens"], j["mask"], 0.125, partition_size=128, workspace=ws)
        # the same workspace: on one stream the calls follow each other
        return (a, *pa.verify_drafts(j["logits"], j["toks"], j["uni"], j["par"], workspace=ws))

    want = [[t.clone() for t in run(j, False)] for j in jobs]
    streams, graphs, held = [torch.cuda.Stream() for _ in jobs], [], []
    for j, s in zip(jobs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run(j, True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            held.append(run(j, True))
        graphs.append(graph)
    for _ in range(6):
        torch.cuda.synchronize()
        for outs in held:
            for t in outs:
                t.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
        # and eager calls on two more streams meanwhile: each stream has its own shared workspace
        others = [torch.cuda.Stream() for _ in jobs]
        eager = []
        for j, s in zip(jobs, others):
            with torch.cuda.stream(s):
                eager.append(run(j, False))
        torch.cuda.synchronize()
        for w, h, e in zip(want, held, eager):
            for x, y, z in zip(w, h, e):
                assert torch.equal(x, y) and torch.equal(x, z)


def test_a_capture_whose_workspace_was_not_reserved_raises(pa, gpu):
    logits = torch.zeros(64, 16, 20001, dtype=torch.float16, device=gpu)
    toks = torch.zeros(64, 16, dtype=torch.int64, device=gpu)
    from ai_infra_train_infer_amd import attention
    kept = dict(attention._WORKSPACES)
    attention._WORKSPACES.clear()
    try:
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="workspace"):
            with torch.cuda.graph(graph):
                pa.verify_drafts(logits, toks, temperature=0.0)
    finally:
        attention._WORKSPACES.update(kept)
    torch.cuda.synchronize()
    assert pa.verify_drafts(logits, toks, temperature=0.0)[1].min() >= 1


@pytest.mark.parametrize("pad", [-1, 1 << 40])
def test_padding_ids_never_reach_the_model(pa, gpu, pad):
    """Ids behind a row's nodes that no vocabulary holds, as verify_drafts writes them: the other rows' logits and the cache
    are those of a step padded with ordinary ids."""
    rng = random.Random(13)
    model = small_model(pa)
    sess = Speculating(pa, model, gpu)
    sess.start([[rng.randrange(512) for _ in range(n)] for n in (20, 33, 5)])
    nodes, real = 6, [6, 0, 3]
    par, num = i32([make_parents("tree", nodes, rng) for _ in real], gpu), i32(real, gpu)
    tables, ctx = sess.tables(nodes, gpu), i32(sess.lens(), gpu)
    toks = torch.tensor([[rng.randrange(512) for _ in range(nodes)] for _ in real], device=gpu)
    odd = toks.clone()
    for b, n in enumerate(real):
        odd[b, n:] = pad
        toks[b, n:] = 0
    cache = sess.pool.kv_cache_tensor
    before = cache.clone()
    want = sess.runner.run_drafts(toks, par, tables, ctx, num_nodes=num)
    after = cache.clone()
    cache.copy_(before)
    got = sess.runner.run_drafts(odd, par, tables, ctx, num_nodes=num)
    assert torch.equal(cache, after) and got.shape == want.shape
    for b, n in enumerate(real):
        assert torch.equal(got[b, :n], want[b, :n])


@pytest.mark.parametrize("cache_dtype", ["fp16", "fp8"])
def test_a_captured_steps_cache_is_that_of_its_own_path(pa, gpu, cache_dtype):
    """After a replay the cache holds, bit for bit, what was there but in the places of the drafted nodes, and in these the rows
    of an eager forward committed along the replay's own path and counts (fp16: as close as two forwards are; their products
    may be cut differently)."""
    from ai_infra_train_infer_amd.attention import sizing_graph_workspace
    rng = random.Random(17)
    model = small_model(pa, cache_dtype)
    sess = Speculating(pa, model, gpu, cache_dtype=cache_dtype)
    sess.start([[rng.randrange(512) for _ in range(n)] for n in (30, 9, 50, 3)])
    nodes = 10
    tables, ctx = sess.tables(nodes, gpu), i32(sess.lens(), gpu)
    toks = torch.zeros(4, nodes, dtype=torch.int64, device=gpu)
    par, num = i32([make_parents("tree", nodes, rng) for _ in range(4)], gpu), i32([nodes] * 4, gpu)
    cache = sess.pool.kv_cache_tensor

    def step():
        logits = sess.runner.run_drafts(toks, par, tables, ctx, num_nodes=num)
        out = pa.verify_drafts(logits, toks, parents=par, num_nodes=num, temperature=0.0)
        return (*out, sess.pool.commit_drafts(tables, ctx, out[2], out[1]))

    start = cache.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), sizing_graph_workspace():
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    kept = 0
    for replay in range(4):
        torch.cuda.synchronize()
        par.copy_(torch.tensor([make_parents(rng.choice(["tree", "deep", "star"]), nodes, rng) for _ in range(4)]))
        num.copy_(torch.tensor([nodes, rng.randrange(nodes + 1), 4, nodes]))
        toks.copy_(torch.tensor([[rng.randrange(512) for _ in range(nodes)] for _ in range(4)]))
        cache.copy_(start)
        first = sess.runner.run_drafts(toks, par, tables, ctx, num_nodes=num).float()
        for b in range(4):                                 # the last child of the root is the target's choice
            children = [c for c in range(1, nodes) if int(par[b, c]) == 0]
            toks[b, children[-1]] = int(first[b, 0].argmax())
        cache.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        got, (out, counts, path, after) = cache.clone(), (t.clone() for t in held)
        kept += int((counts - 1).clamp(min=0).sum())
        cache.copy_(start)
        sess.runner.run_drafts(toks, par, tables, ctx, num_nodes=num)
        assert torch.equal(sess.pool.commit_drafts(tables, ctx, path, counts), after) and torch.equal(after, ctx + counts)
        drafted = torch.zeros(cache.shape[2:4], dtype=torch.bool, device=gpu)
        for b in range(4):
            for i in range(int(num[b])):
                p = int(ctx[b]) + i
                drafted[tables[b, p // 16], p % 16] = True
        for x in (got, cache):
            assert torch.equal(x.view(torch.uint8).view(*x.shape[:4], -1)[:, :, ~drafted],
                               start.view(torch.uint8).view(*x.shape[:4], -1)[:, :, ~drafted])
        if cache_dtype == "fp16":
            torch.testing.assert_close(got[:, :, drafted].float(), cache[:, :, drafted].float(), rtol=2e-2, atol=2e-2)
    assert kept >= 6        # paths of more than the root were committed
