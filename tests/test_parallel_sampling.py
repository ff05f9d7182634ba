"""Several continuations of one prompt: forked block tables, the plain restatements of the operators, and the engine path
(torch and C++ backends on CPU, native kernels on the GPU)."""
import math

import pytest
import torch

from mod_b200.engine.block_manager import BlockManager, PrefixCachingBlockManager
from mod_b200.engine.parallel_sampling import ParallelSampler
from mod_b200.engine.sequence import SamplingParams, Sequence
from mod_b200.ops import reference as R


def _prompts():
    g = torch.Generator().manual_seed(5)
    base = torch.randint(1, 500, (12,), generator=g).tolist()
    return [base * 3, (base[:5] + [7, 8]) * 4, list(range(3, 30)), [9] * 16]


def _engine(backend="torch", device="cpu", name="tiny-dense", fp32=True, **kw):
    from mod_b200.config import get_preset
    from mod_b200.engine.llm_engine import LLMEngine
    from mod_b200.models.weights import random_weights

    cfg = get_preset(name)
    w = random_weights(cfg, device=device, dtype=torch.float32, seed=0) if fp32 else None
    return LLMEngine(cfg, weights=w, backend=backend, device=device, max_batch=16, max_model_len=160, use_graphs=False, **kw)


# ------------------------------------------------------------------ block tables
@pytest.mark.parametrize("mgr", [BlockManager, PrefixCachingBlockManager])
@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 48, 50])
def test_fork_shares_full_blocks(mgr, tokens):
    m = mgr(32, 16, max_seqs=8)
    p = Sequence(prompt=list(range(tokens)))
    assert m.allocate(p, tokens)
    p.num_cached = tokens
    if mgr is PrefixCachingBlockManager:
        m.register(p)
    kids = [Sequence(prompt=list(p.prompt)) for _ in range(3)]
    full, part = divmod(tokens, 16)
    for c in kids:
        pairs = m.fork(p, c)
        assert c.blocks[:full] == p.blocks[:full] and c.num_cached == tokens
        assert pairs == ([(p.blocks[full], c.blocks[full])] if part else [])
    last = [c.blocks[full] for c in kids if part] + ([p.blocks[full]] if part else [])
    assert len(set(last)) == len(last)
    assert m.num_free == 32 - full - len(last)
    m.release(p)
    assert m.num_free == 32 - full - 3 * bool(part)          # the children still hold the shared blocks
    for c in kids[:2]:
        m.release(c)
    assert m.num_free == 32 - full - bool(part)
    m.release(kids[2])
    assert m.num_free == 32 and not m.owners
    # and the freed blocks can all be taken again
    s = Sequence(prompt=[1000 + i for i in range(32 * 16)])
    assert m.allocate(s, 32 * 16) and sorted(s.blocks) == list(range(32))


def test_fork_without_room():
    m = BlockManager(2, 16, max_seqs=2)
    p, c = Sequence(prompt=list(range(20))), Sequence(prompt=list(range(20)))
    assert m.allocate(p, 20)
    p.num_cached = 20
    assert m.fork(p, c) is None and c.blocks == [] and not m.owners
    m = BlockManager(4, 16, max_seqs=1)
    assert m.allocate(p2 := Sequence(prompt=[1]), 1)
    p2.num_cached = 1
    assert m.fork(p2, Sequence(prompt=[1])) is None


def test_moved_keeps_owners_and_free_blocks():
    m = BlockManager(8, 16, max_seqs=4)
    a, b = Sequence(prompt=[0] * 16), Sequence(prompt=[0] * 16)
    filler = Sequence(prompt=[0] * 48)
    assert m.allocate(filler, 48) and m.allocate(a, 16)
    a.num_cached = 16
    assert m.fork(a, b) == []
    m.release(filler)
    remap = [-1] * 8
    remap[a.blocks[0]] = 0
    m.moved(remap)
    a.blocks = b.blocks = [0]
    a.blocks, b.blocks = [0], [0]
    assert sorted(m.free) == list(range(1, 8))
    m.release(a)
    assert m.num_free == 7
    m.release(b)
    assert m.num_free == 8


# ------------------------------------------------------------------ plain restatements
def test_reference_attn_shared_equals_dense_attention():
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(6, 2, 16, 64, generator=g), torch.randn(6, 2, 64, 16, generator=g)
    tables = torch.tensor([[5, 2, 0], [5, 1, 3]], dtype=torch.int32)
    ctx, cu = torch.tensor([40, 19], dtype=torch.int32), torch.tensor([0, 3, 4], dtype=torch.int32)
    q = torch.randn(4, 4, 64, generator=g)
    out = R.attn_shared(q, k, v, tables, ctx, cu)
    for t, (b, n) in enumerate([(0, 38), (0, 39), (0, 40), (1, 19)]):
        kk, vv = R.gather_kv(k, tables[b], n).double(), R.gather_v(v, tables[b], n).double()
        for h in range(4):
            p = torch.softmax(kk[:, h // 2] @ q[t, h].double() / math.sqrt(64), 0)
            assert torch.allclose(out[t, h].double(), p @ vv[:, h // 2], atol=1e-5)


def test_reference_compact_and_copy():
    k, v = [torch.arange(8.0).view(8, 1, 1, 1).clone()], [-torch.arange(8.0).view(8, 1, 1, 1)]
    tables, lens = torch.tensor([[6, 1, 9], [1, 4, 0]], dtype=torch.int32), torch.tensor([32, 20], dtype=torch.int32)
    out, remap, live = R.kv_compact(k, v, tables, lens)
    assert int(live) == 3 and remap.tolist() == [-1, 1, -1, -1, 0, -1, 2, -1]
    assert out.tolist() == [[2, 1, 0], [1, 0, 0]]
    assert k[0].flatten().tolist()[:3] == [4.0, 1.0, 6.0] and v[0].flatten().tolist()[:3] == [-4.0, -1.0, -6.0]
    R.kv_copy_pages(k, v, torch.tensor([7, -1], dtype=torch.int32), torch.tensor([3, 5], dtype=torch.int32))
    assert k[0].flatten().tolist() == [4.0, 1.0, 6.0, 7.0, 4.0, 5.0, 6.0, 7.0]


def test_reference_verify_follows_the_target():
    B, V = 4000, 5
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(2, V, generator=g)
    q = torch.softmax(torch.randn(V, generator=g), 0)
    p = torch.softmax(logits[0].double(), 0)
    drafts = torch.multinomial(q, B, replacement=True, generator=g)[:, None]
    acc, tok, probs = R.verify_sampled(logits.repeat(B, 1), torch.arange(0, 2 * B + 1, 2, dtype=torch.int32), drafts,
                                       torch.rand(B, 1, generator=g), torch.empty(B, V).exponential_(generator=g),
                                       torch.ones(B), q.expand(B, 1, V))
    first = torch.where(acc == 1, drafts[:, 0], tok)
    f = torch.bincount(first, minlength=V).double() / B
    assert ((f - p).abs() <= 5 * torch.sqrt(p * (1 - p) / B)).all()
    assert torch.allclose(probs[:, 0].double(), p[first], atol=1e-6)


# ------------------------------------------------------------------ engine path
@pytest.mark.parametrize("backend,name", [("torch", "tiny-dense"), ("torch", "tiny-moe"), ("cpu", "tiny-dense")])
@pytest.mark.parametrize("caching", [False, True])
def test_greedy_samples_equal_greedy_decoding(backend, name, caching):
    P = _prompts()
    ref = _engine(backend, name=name).generate(P, SamplingParams(max_new_tokens=20))
    eng = _engine(backend, name=name, prefix_caching=caching)
    s = ParallelSampler(eng, drafts=3)
    got = s.generate(P, 3, SamplingParams(max_new_tokens=20))
    assert got == [[r] * 3 for r in ref]
    assert s.stats.steps > 0 and eng.blocks.num_free == eng.blocks.num_blocks and not eng.blocks.owners
    assert len(eng.blocks.free_slots) == eng.blocks.max_seqs
    assert eng.generate(P, SamplingParams(max_new_tokens=20)) == ref      # the engine goes on as before


def test_seeded_samples_differ_and_repeat():
    p = SamplingParams(max_new_tokens=12, temperature=1.0, seed=4)
    a = _engine().generate_parallel(_prompts()[:2], 4, p)
    b = _engine().generate_parallel(_prompts()[:2], 4, p)
    assert a == b and len({tuple(x) for g in a for x in g}) > 4
    assert all(len(x) == 12 for g in a for x in g)
    c = _engine().generate_parallel(_prompts()[:2], 4, SamplingParams(max_new_tokens=12, temperature=1.0, seed=5))
    assert a != c


def test_filters_keep_to_the_allowed_tokens():
    P = _prompts()[:2]
    ref = _engine().generate(P, SamplingParams(max_new_tokens=10))
    got = _engine().generate_parallel(P, 2, SamplingParams(max_new_tokens=10, temperature=1.5, top_k=1, seed=1))
    assert got == [[r] * 2 for r in ref]


def test_early_ends_compact_the_pool():
    eng = _engine()
    ref = _engine().generate(_prompts(), SamplingParams(max_new_tokens=24))
    calls = []
    keep = eng.compact_kv
    eng.compact_kv = lambda extra=None: calls.append(keep(extra)) or calls[-1]
    # each prompt's stop token comes at its own time, so that most sequences end before the others
    eos = ref[0][2]
    got = eng.generate_parallel(_prompts(), 3, SamplingParams(max_new_tokens=24, eos_token_id=eos))
    want = [r[:r.index(eos) + 1] if eos in r else r for r in ref]
    assert got == [[w] * 3 for w in want]
    assert calls and eng.blocks.num_free == eng.blocks.num_blocks


def test_compact_kv_between_steps():
    P, params = _prompts(), SamplingParams(max_new_tokens=16)
    ref = _engine().generate(P, params)
    for caching in (False, True):
        eng = _engine(prefix_caching=caching)
        ids = [eng.add_request(p, params) for p in P]
        eng.step()
        eng.abort(ids[1])
        eng.step()
        live = eng.compact_kv()
        used = {b for s in eng.scheduler.running for b in s.blocks}
        assert used == set(range(live)) and eng.blocks.num_free == eng.blocks.num_blocks - live
        while eng.has_unfinished():
            eng.step()
        assert [eng.seqs[i].output for i in (ids[0], *ids[2:])] == [ref[0], *ref[2:]]


def test_refuses():
    with pytest.raises(ValueError):
        ParallelSampler(_engine(name="tiny-next", fp32=False))
    s = ParallelSampler(_engine())
    for prompts, n in (([[1, 2]], 0), ([[1, 2]], 16), ([[]], 2), ([[1] * 150], 2)):
        with pytest.raises(ValueError):
            s.generate(prompts, n, SamplingParams(max_new_tokens=16))
    eng = _engine(num_blocks=4)
    with pytest.raises(RuntimeError, match="exhausted"):
        eng.generate_parallel([list(range(1, 41))], 4, SamplingParams(max_new_tokens=8))
    assert eng.blocks.num_free == 4 and not eng.blocks.owners


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["tiny-dense", "tiny-moe", "tiny-glm"])
def test_native_greedy_samples(name):
    P = _prompts()
    ref = _engine("native", "cuda:0", name, fp32=False).generate(P, SamplingParams(max_new_tokens=24))
    eng = _engine("native", "cuda:0", name, fp32=False)
    s = ParallelSampler(eng, drafts=4)
    assert s.shared
    got = s.generate(P, 3, SamplingParams(max_new_tokens=24))
    # The one-token and the multi-token paths round differently: where a continuation leaves the greedy one, the two
    # tokens' logits have to tie, within two bf16 roundings (2^-8 each) in each of the two paths.
    for prompt, r, g in zip(P, ref, got):
        for x in g:
            k = next((i for i in range(24) if x[i] != r[i]), None)
            if k is None:
                continue
            q = Sequence(prompt=prompt + r[:k], params=SamplingParams())
            assert eng.blocks.allocate(q, q.length)
            logits = eng.runner.prefill([q], [q.length], return_logits=True)[0]
            eng.blocks.release(q)
            top = float(logits.max())
            assert min(float(logits[x[k]]), float(logits[r[k]])) >= top - 2 ** -6 * float(logits.abs().max()), (k, x, r)
    assert eng.blocks.num_free == eng.blocks.num_blocks
    from mod_b200.ops import check_status

    torch.cuda.synchronize()
    check_status()


@pytest.mark.gpu
def test_native_samples_repeat():
    p = SamplingParams(max_new_tokens=16, temperature=0.8, top_p=0.9, seed=3)
    a = _engine("native", "cuda:0", fp32=False).generate_parallel(_prompts(), 3, p)
    b = _engine("native", "cuda:0", fp32=False).generate_parallel(_prompts(), 3, p)
    assert a == b and all(len(x) == 16 for g in a for x in g)


@pytest.mark.gpu
def test_native_compact_kv_with_captured_steps():
    from mod_b200.config import get_preset
    from mod_b200.engine.llm_engine import LLMEngine

    P, params = _prompts(), SamplingParams(max_new_tokens=16)
    mk = lambda: LLMEngine(get_preset("tiny-dense"), backend="native", device="cuda:0", max_batch=16, max_model_len=160)  # noqa: E731
    ref = mk().generate(P, params)
    eng = mk()
    ids = [eng.add_request(p, params) for p in P]
    for _ in range(3):
        eng.step()
    eng.abort(ids[0])
    live = eng.compact_kv()
    assert {b for s in eng.scheduler.running for b in s.blocks} == set(range(live))
    while eng.has_unfinished():
        eng.step()
    assert [eng.seqs[i].output for i in ids[1:]] == ref[1:]
