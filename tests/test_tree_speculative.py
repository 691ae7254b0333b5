"""Speculative decoding with trees of drafts and with sampling: the same tokens as without drafts, whatever the drafts are; min-p; batches built from page lists."""
import dataclasses

import pytest
import torch

from gemm_b200 import _native
from gemm_b200.models import reference
from gemm_b200.models.config import get_config
from gemm_b200.models.transformer import ForwardBatch, KvCache, Transformer
from gemm_b200.models.weights import synthetic_weights
from gemm_b200.ops import paging, sampling, tree
from gemm_b200.serve.engine import Engine, SamplingParams
from gemm_b200.serve.llm import LLM
from gemm_b200.serve.speculative import CallableDrafter, NgramTreeDrafter, SpeculativeDecoder

gpu = pytest.mark.gpu


def decoder(name, drafter, device="cpu", page=16, n_pages=96):
    cfg = get_config(name)
    w = synthetic_weights(cfg, "bf16", device="cpu", seed=3)
    kv = KvCache.allocate(cfg, n_pages, page, device)
    return cfg, SpeculativeDecoder(Transformer(w if device == "cpu" else w.to(device), kv), kv, page, n_pages, drafter)


class KnowingTrees:
    """Trees with the right continuation in one branch (as far as ``known`` goes), wrong ones beside it, and the right token twice among siblings."""

    def __init__(self, known, gamma=4, vocab=512):
        self.known, self.gamma, self.vocab = known, gamma, vocab

    def propose_tree(self, tokens):
        good = next((f[len(tokens): len(tokens) + self.gamma] for f in self.known if list(tokens) == f[: len(tokens)]), [])
        toks, parents, at = [], [], -1
        for x in good:
            toks += [(x + 1) % self.vocab, x, x]                            # a wrong sibling, the right token, and again
            parents += [at, at, at]
            toks.append((x + 2) % self.vocab)                               # a child of the wrong sibling
            parents.append(len(toks) - 4)
            at = len(toks) - 3
        return toks, parents


def test_tree_drafter():
    d = NgramTreeDrafter(gamma=3, width=2, max_ngram=2)
    assert d.propose_tree([5, 6, 7, 8, 5, 6, 7, 9, 5, 6]) == ([7, 9, 5, 8, 5], [-1, 0, 1, 0, 3])
    assert d.propose_tree([1, 2, 3]) == ([], [])
    assert NgramTreeDrafter(gamma=2, width=8).propose_tree([4, 4, 4])[0] == [4]
    for bad in (dict(gamma=0), dict(width=0), dict(gamma=64, width=4)):
        with pytest.raises(ValueError):
            NgramTreeDrafter(**bad)


@pytest.mark.parametrize("sp", [SamplingParams(), SamplingParams(temperature=0.8, top_k=40, top_p=0.9, seed=5), SamplingParams(temperature=1.2, min_p=0.05, seed=9)])
def test_trees_equal_no_drafts(sp):
    torch.manual_seed(1)
    cfg, plain = decoder("tiny-dense", None)
    prompts = [torch.randint(0, cfg.vocab, (n,)).tolist() for n in (21, 9, 40)]
    n_new = 14
    ref = plain.generate(prompts, n_new, sp=sp)
    if sp.temperature > 0:
        assert ref == decoder("tiny-dense", None)[1].generate(prompts, n_new, sp=sp)
        assert ref != plain.generate(prompts, n_new, sp=dataclasses.replace(sp, seed=sp.seed + 1))
    known = [p + o for p, o in zip(prompts, ref)]
    dec = decoder("tiny-dense", KnowingTrees(known))[1]
    assert dec.generate(prompts, n_new, sp=sp) == ref
    assert dec.stats.verify_steps == 3 and dec.stats.tokens_per_step > 10               # 1 + 5 + 5 + 3 tokens
    half = KnowingTrees([k[:len(k) - 6] for k in known])
    assert decoder("tiny-dense", half)[1].generate(prompts, n_new, sp=sp) == ref
    assert decoder("tiny-dense", NgramTreeDrafter(gamma=3, width=3))[1].generate(prompts, n_new, sp=sp) == ref
    chain = CallableDrafter(lambda t: next((f[len(t): len(t) + 4] for f in known if list(t) == f[: len(t)]), [7, 7]), gamma=4)
    assert decoder("tiny-dense", chain)[1].generate(prompts, n_new, sp=sp) == ref
    stop = ref[0][5]
    got = decoder("tiny-dense", KnowingTrees(known))[1].generate(prompts, n_new, stop_token_ids=[stop], sp=sp)
    assert got == [r[: r.index(stop) + 1] if stop in r else r for r in ref]
    # a cache with no room for drafts: one token a step
    need = sum((len(p) + n_new + 1 + 15) // 16 for p in prompts)
    tight = decoder("tiny-dense", KnowingTrees(known), n_pages=need)[1]
    assert tight.generate(prompts, n_new, sp=sp) == ref


def test_llm_and_refusals():
    torch.manual_seed(2)
    cfg = get_config("tiny-dense")
    w = synthetic_weights(cfg, "bf16", device="cpu", seed=3)
    mk = lambda: LLM(w, None, max_running=4, num_pages=64, page_size=16)          # noqa: E731
    prompts = [torch.randint(0, cfg.vocab, (n,)).tolist() for n in (12, 30)]
    want = mk().generate(prompts, SamplingParams(max_new_tokens=9))
    got, stats = mk().generate_speculative(prompts, 9, drafter=NgramTreeDrafter(gamma=3, width=2))
    assert got == want and stats.produced == 2 * 8
    sp = SamplingParams(max_new_tokens=9, temperature=0.9, top_p=0.9, min_p=0.02, seed=4)
    a, b = mk().generate(prompts, sp), mk().generate(prompts, sp)
    assert a == b and all(0 <= t < cfg.vocab for o in a for t in o)
    one = mk().generate(prompts, dataclasses.replace(sp, min_p=1.0))              # only the likeliest token is as likely as itself
    assert one == want
    assert Engine(w, 4, 64, page_size=16).generate(prompts, dataclasses.replace(sp, min_p=1.0)) == want
    assert Engine(w, 4, 64, page_size=16).generate(prompts, sp) == Engine(w, 4, 64, page_size=16).generate(prompts, sp)
    hybrid = get_config("tiny-qwen35")
    wh = synthetic_weights(hybrid, "bf16", device="cpu", seed=3)
    kv = KvCache.allocate(hybrid, 16, 16, "cpu")
    with pytest.raises(ValueError):
        SpeculativeDecoder(Transformer(wh, kv), kv, 16, 16, NgramTreeDrafter())
    fb = ForwardBatch.build_tree([0], [[1, 2]], [[-1, 0]], [[0]], 16, "cpu")
    with pytest.raises(NotImplementedError):
        Transformer(wh, kv).forward(fb)
    for bad in (([0], [[1, 2]], [[-1]], [[0]]), ([0], [[1, 2]], [[-1, 1]], [[0]]), ([0], [[1, 2]], [[0, 0]], [[0]]), ([0], [[]], [[]], [[0]]),
                ([0], [[1] * 257], [[-1] + [0] * 256], [list(range(20))])):
        with pytest.raises(ValueError):
            ForwardBatch.build_tree(*bad, 16, "cpu")
    with pytest.raises(IndexError):
        ForwardBatch.build_tree([15], [[1, 2]], [[-1, 0]], [[0]], 16, "cpu")


def test_uniform_numbers():
    u = sampling.uniform_numbers(3, 7, 5000)
    assert u.min() >= 0 and u.max() < 1 and abs(float(u.mean()) - 0.5) < 0.02 and len(set(u.tolist())) > 4990
    assert sampling.uniform_numbers(3, 7, 1)[0] == u[0] and sampling.uniform_numbers(4, 7, 1)[0] != u[0] and sampling.uniform_numbers(3, 8, 1)[0] != u[0]


@gpu
def test_build_paged_equals_build():
    torch.manual_seed(0)
    for q, ctx, page in (([1, 1, 1], [5, 16, 31], 16), ([30, 1, 0, 77], [0, 100, 3, 51], 32), ([3], [0], 128)):
        have = [(a + b + page - 1) // page for a, b in zip(q, ctx)]
        ids = torch.randperm(sum(have) + 2).tolist()
        pages = [ids[sum(have[:i]): sum(have[:i + 1])] for i in range(len(q))]
        bt = torch.zeros(len(q), max(have), dtype=torch.int32)
        for i, p in enumerate(pages):
            bt[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
        toks = list(range(sum(q)))
        slots = [7 + i for i in range(len(q))]
        want = ForwardBatch.build(q, ctx, toks, bt, page, 8, 2, "cuda", seq_slots=slots)
        got = ForwardBatch.build_paged(q, ctx, toks, pages, page, 8, 2, "cuda", seq_slots=slots)
        for f in dataclasses.fields(ForwardBatch):
            a, b = getattr(got, f.name), getattr(want, f.name)
            assert torch.equal(a, b) and a.dtype == b.dtype if torch.is_tensor(a) else a == b, f.name
        assert torch.equal(ForwardBatch.build_paged(q, ctx, toks, pages, page, 8, 2, "cuda", rows=[0, 2] if sum(q) > 2 else [0]).logit_rows.cpu(),
                           torch.tensor([0, 2] if sum(q) > 2 else [0]))
    with pytest.raises(IndexError):
        ForwardBatch.build_paged([10], [250], list(range(10)), [[0, 1]], 128, 8, 2, "cuda")


@gpu
def test_verification_step_equals_its_parts():
    """Tables, attention, draws and commit in a row on the GPU against the same calls on the CPU: one sequence of operators as a verification step makes it."""
    from tests.test_tree_ops import commit_inputs
    from gemm_b200.ops import paging
    nodes, ctx, page, hq, hkv, d, v = [12, 1, 30], [200, 0, 77], 16, 8, 2, 64, 300
    s = commit_inputs(nodes, ctx, page, [((hkv, d), torch.bfloat16)] * 4, seed=3, accept=0.9, vocab=40)
    need = [(a + b + page - 1) // page for a, b in zip(nodes, ctx)]
    pages = [s["block_table"][i, :n].tolist() for i, n in enumerate(need)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)                     # noqa: E731
    args = (i32(nodes), i32(ctx), i32([0] + list(torch.tensor(need).cumsum(0))), i32([x for p in pages for x in p]), page, sum(nodes), max(need), s["parents"], max(nodes))
    g = torch.Generator().manual_seed(0)
    caches = [(torch.randn(c.shape, generator=g)).bfloat16() for c in s["caches"]]
    q = (torch.randn(sum(nodes), hq, d, generator=g) * 0.2).bfloat16()
    head = torch.randn(hq * d, v, generator=g) * 0.3
    u = torch.rand(sum(nodes), generator=g)
    res = []
    for dev in ("cpu", "cuda"):
        mv = lambda x: x.to(dev)                                           # noqa: E731,B023
        t = paging.batch_tables(*[mv(a) if torch.is_tensor(a) else a for a in args])
        cs = [mv(c).clone() for c in caches]
        o = tree.tree_attention(mv(q), cs[0], cs[1], t.cu_q, t.kv_len, t.block_table, page, t.mask, max(nodes))
        # (the same logits on both sides: what is compared here is that the parts fit, not their rounding)
        logits = mv(res[0]["logits"]) if res else o.float().reshape(sum(nodes), -1) @ head
        drawn = sampling.draw(logits, mv(u), 0.8, 20, 0.9, 0.01)
        drawn = torch.where(mv(torch.arange(sum(nodes)) % 3 == 0), drawn, mv(s["sampled"]))              # most of the drafts' own tokens, so that paths are long
        acc = tree.tree_commit(cs, mv(s["tokens"]), mv(s["parents"]), drawn, t.cu_q, t.kv_len, t.block_table, page, max(nodes))
        res.append(dict(t=t, o=o, logits=logits, drawn=drawn, acc=acc, cs=cs))
    a, b = res
    for x, y in zip(list(a["t"]) + list(a["acc"]) + a["cs"] + [a["drawn"]], list(b["t"]) + list(b["acc"]) + b["cs"] + [b["drawn"]]):
        assert torch.equal(x, y.cpu())
    assert (a["o"].float() - b["o"].float().cpu()).abs().max() < 2 ** -6
    assert int(a["acc"].count.max()) > 1


@gpu
@pytest.mark.parametrize("name", ["tiny-dense", "tiny-moe"])
def test_trees_on_gpu(name):
    """Every token is a legitimate greedy choice of the fp32 oracle, and known continuations are accepted several at a time."""
    torch.manual_seed(4)
    cfg, plain = decoder(name, None, "cuda")
    w_cpu = synthetic_weights(cfg, "bf16", device="cpu", seed=3)
    prompts = [torch.randint(0, cfg.vocab, (n,)).tolist() for n in (33, 70)]
    ref = plain.generate(prompts, 12)
    dec = decoder(name, KnowingTrees([p + o for p, o in zip(prompts, ref)]), "cuda")[1]
    out = dec.generate(prompts, 12)
    _native.assert_status_ok()
    for p, o in zip(prompts, out):
        logits = reference.reference_logits(w_cpu, torch.tensor(list(p) + list(o))[:-1]).float()
        for j, tok in enumerate(o):
            row = logits[len(p) - 1 + j]
            assert row[tok] >= row.max() - 0.3 * row.std()
    assert dec.stats.tokens_per_step > 2.0
    sp = SamplingParams(temperature=0.8, top_k=30, top_p=0.9, min_p=0.02, seed=2)
    a = decoder(name, NgramTreeDrafter(gamma=3, width=3), "cuda")[1].generate(prompts, 12, sp=sp)
    assert all(len(o) == 12 and all(0 <= t < cfg.vocab for t in o) for o in a)
    _native.assert_status_ok()


@gpu
def test_engine_min_p_on_gpu():
    """A decode loop replayed from a graph draws with new numbers at every step, the same as an eager one."""
    cfg = get_config("tiny-dense")
    w = synthetic_weights(cfg, "bf16", device="cpu", seed=3).to("cuda")
    prompts = [[5, 6, 7, 8], [9, 3, 1]]
    sp = SamplingParams(max_new_tokens=12, temperature=1.5, min_p=0.001, seed=7)
    a = Engine(w, 2, 64, page_size=16).generate(prompts, sp, use_graph=True)
    b = Engine(w, 2, 64, page_size=16).generate(prompts, sp, use_graph=False)
    assert a == b and len(set(a[0])) > 3


def windowed(drafter, device):
    cfg = dataclasses.replace(get_config("tiny-dense"), sliding_window=10)
    w = synthetic_weights(cfg, "bf16", device="cpu", seed=3)
    kv = KvCache.allocate(cfg, 96, 16, device)
    return cfg, w, SpeculativeDecoder(Transformer(w if device == "cpu" else w.to(device), kv), kv, 16, 96, drafter)


def test_trees_with_a_sliding_window():
    """Branches of several depths, each with a window of its own."""
    torch.manual_seed(2)
    cfg, _, plain = windowed(None, "cpu")
    prompts = [torch.randint(0, cfg.vocab, (n,)).tolist() for n in (5, 33)]
    ref = plain.generate(prompts, 16)
    assert ref != decoder("tiny-dense", None)[1].generate(prompts, 16)
    dec = windowed(KnowingTrees([p + o for p, o in zip(prompts, ref)], gamma=6), "cpu")[2]
    assert dec.generate(prompts, 16) == ref and dec.stats.tokens_per_step > 8


@gpu
def test_trees_with_a_sliding_window_on_gpu():
    torch.manual_seed(2)
    cfg, w, plain = windowed(None, "cuda")
    prompts = [torch.randint(0, cfg.vocab, (n,)).tolist() for n in (5, 33)]
    dec = windowed(KnowingTrees([p + o for p, o in zip(prompts, plain.generate(prompts, 16))], gamma=6), "cuda")[2]
    out = dec.generate(prompts, 16)
    _native.assert_status_ok()
    for p, o in zip(prompts, out):
        logits = reference.reference_logits(w, torch.tensor(list(p) + list(o))[:-1]).float()
        for j, tok in enumerate(o):
            row = logits[len(p) - 1 + j]
            assert row[tok] >= row.max() - 0.3 * row.std()
    assert dec.stats.tokens_per_step > 2.0


@pytest.mark.parametrize("window,gamma", [(1, 3), (4, 9), (10, 12)])
@pytest.mark.parametrize("sp", [SamplingParams(), SamplingParams(temperature=0.8, top_k=40, top_p=0.9, seed=5)])
def test_trees_deeper_than_the_window(window, gamma, sp):
    """Drafts that reach past the window, as a tree and as a sampled chain: the tokens of decoding without drafts, all drafts accepted."""
    def make(drafter):
        cfg = dataclasses.replace(get_config("tiny-dense"), sliding_window=window)
        kv = KvCache.allocate(cfg, 96, 16, "cpu")
        return SpeculativeDecoder(Transformer(synthetic_weights(cfg, "bf16", device="cpu", seed=3), kv), kv, 16, 96, drafter)
    torch.manual_seed(2)
    prompts = [torch.randint(0, 512, (n,)).tolist() for n in (5, 33)]
    ref = make(None).generate(prompts, 16, sp=sp)
    known = [p + o for p, o in zip(prompts, ref)]
    dec = make(KnowingTrees(known, gamma=gamma))
    assert dec.generate(prompts, 16, sp=sp) == ref and dec.stats.verify_steps == -(-15 // (gamma + 1))
    chain = CallableDrafter(lambda t: next((f[len(t): len(t) + gamma] for f in known if list(t) == f[: len(t)]), [7, 7]), gamma=gamma)
    assert make(chain).generate(prompts, 16, sp=sp) == ref


@gpu
def test_trees_deeper_than_the_window_on_gpu():
    """Every token is a legitimate greedy choice of the fp32 oracle, with branches of three windows' length."""
    torch.manual_seed(2)
    cfg = dataclasses.replace(get_config("tiny-dense"), sliding_window=4)
    w = synthetic_weights(cfg, "bf16", device="cpu", seed=3).to("cuda")

    def make(drafter):
        kv = KvCache.allocate(cfg, 96, 16, "cuda")
        return SpeculativeDecoder(Transformer(w, kv), kv, 16, 96, drafter)
    prompts = [torch.randint(0, cfg.vocab, (n,)).tolist() for n in (5, 33)]
    dec = make(KnowingTrees([p + o for p, o in zip(prompts, make(None).generate(prompts, 24))], gamma=12))
    out = dec.generate(prompts, 24)
    _native.assert_status_ok()
    for p, o in zip(prompts, out):
        logits = reference.reference_logits(w, torch.tensor(list(p) + list(o))[:-1]).float()
        for j, tok in enumerate(o):
            row = logits[len(p) - 1 + j]
            assert row[tok] >= row.max() - 0.3 * row.std()
    assert dec.stats.tokens_per_step > 4.0


@pytest.mark.parametrize("name", ["tiny-qwen35", "tiny-fidolix"])
def test_every_forward_refuses_trees_on_other_models(name):
    """Recurrent layers would take siblings for a chain."""
    cfg = get_config(name)
    kv = KvCache.allocate(cfg, 16, 16, "cpu")
    m = Transformer(synthetic_weights(cfg, "bf16", device="cpu", seed=3), kv)
    fb = ForwardBatch.build_tree([0], [[1, 2, 3]], [[-1, 0, 0]], [[0]], 16, "cpu")
    for call in (m.forward, m.forward_greedy, m.forward_hidden, lambda b: m.forward_hidden(b, 0, 1)):
        with pytest.raises(NotImplementedError):
            call(fb)


def test_build_tree_refuses_negative_contexts():
    for ctx in ([-1], [4, -2]):
        n = len(ctx)
        with pytest.raises(ValueError):
            ForwardBatch.build_tree(ctx, [[1, 2]] * n, [[-1, 0]] * n, [[0]] * n, 16, "cpu")
    for bad in (dict(ctx_lens=[0]), dict(parents=[[-1, 0]]), dict(pages=[[0]]), dict(parents=[[-1, 0]] * 3)):
        with pytest.raises(ValueError):
            ForwardBatch.build_tree(**{**dict(ctx_lens=[0, 0], tokens=[[1, 2]] * 2, parents=[[-1, 0]] * 2, pages=[[0], [1]], page_size=16, device="cpu"), **bad})


def test_sequential_min_p_above_one():
    """A min-p above 1 counts as 1, as in ``sampling.draw``: the likeliest token alone."""
    from gemm_b200.serve.sequential import SequentialLLM
    x = torch.randn(1, 50, generator=torch.Generator().manual_seed(0))
    for min_p in (1.0, 1.5, 40.0):
        for top_p in (1.0, 0.5):
            sp = SamplingParams(temperature=0.7, top_p=top_p, min_p=min_p)
            assert SequentialLLM._pick(None, x, sp, 0) == int(x.argmax()) == int(sampling.draw(x, torch.tensor([0.5]), 0.7, 0, top_p, min_p)[0])


@gpu
def test_build_paged_of_more_sequences_than_the_table_kernel_takes():
    """A step of any number of sequences is assembled, as ``build`` does it."""
    n = paging.MAX_SEQS + 300
    q, ctx = [1 + i % 3 for i in range(n)], [i % 40 for i in range(n)]
    have = [(a + b + 15) // 16 for a, b in zip(q, ctx)]
    at = [0] + torch.tensor(have).cumsum(0).tolist()
    pages = [list(range(at[i], at[i + 1])) for i in range(n)]
    bt = torch.zeros(n, max(have), dtype=torch.int32)
    for i, p in enumerate(pages):
        bt[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
    want = ForwardBatch.build(q, ctx, list(range(sum(q))), bt, 16, 8, 2, "cuda")
    for count in (paging.MAX_SEQS, n):
        got = ForwardBatch.build_paged(q[:count], ctx[:count], list(range(sum(q[:count]))), pages[:count], 16, 8, 2, "cuda", rows=[3, 0])
        t = sum(q[:count])
        for name, x in (("ids", t), ("positions", t), ("slots", t), ("cu_q", count + 1), ("kv_len", count), ("block_table", count), ("seq_slots", count)):
            a, b = getattr(got, name), getattr(want, name)[:x]
            assert torch.equal(a, b) and a.dtype == b.dtype, name
        assert got.logit_rows.tolist() == [3, 0] and got.logit_rows.is_cuda and got.n_tokens == t


def test_engine_min_p_with_ranks_that_hold_the_whole_head():
    """Tensor-parallel ranks with an unsharded LM head draw alike, each for itself; a share of the vocabulary is refused."""
    cfg = get_config("tiny-dense")
    e = Engine(synthetic_weights(cfg, "bf16", device="cpu", seed=3), 2, 64, page_size=16)
    logits = torch.randn(2, cfg.vocab, generator=torch.Generator().manual_seed(0))
    sp = SamplingParams(temperature=1.3, min_p=0.01, seed=5)
    want = e._sample(logits, sp, 3)

    class Ranks:
        def merge_sampled(self, tok, logits):
            raise AssertionError("there is nothing to merge")
    e.par = Ranks()
    assert torch.equal(e._sample(logits, sp, 3), want)
    with pytest.raises(NotImplementedError):
        e._sample(logits[:, :256].contiguous(), sp, 3)
