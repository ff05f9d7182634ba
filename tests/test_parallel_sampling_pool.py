"""Several continuations of one prompt in an engine that has other work, little room or trouble."""
import pytest
import torch

from mod_b200.engine.parallel_sampling import ParallelSampler
from mod_b200.engine.sequence import SamplingParams
from tests.test_parallel_sampling import _engine, _prompts


def whole(eng):
    return (eng.blocks.num_free == eng.blocks.num_blocks and not eng.blocks.owners
            and len(eng.blocks.free_slots) == eng.blocks.max_seqs)


# ------------------------------------------------------------------ a kernel that gives up
def test_status_is_read_every_step(monkeypatch):
    from mod_b200.engine import parallel_sampling as M

    seen = []
    monkeypatch.setattr(M, "check_status", lambda dev: seen.append(dev))
    eng = _engine()
    s = ParallelSampler(eng)
    s.native = True               # as on the GPU, with the plain operators in the kernels' place
    from mod_b200.ops import reference

    eng.backend.N = reference
    s.generate(_prompts()[:2], 2, SamplingParams(max_new_tokens=6))
    assert len(seen) == s.stats.steps + 1

    def fail(dev):
        raise RuntimeError("mbarrier wait timed out")

    monkeypatch.setattr(M, "check_status", fail)
    with pytest.raises(RuntimeError, match="timed out"):
        s.generate(_prompts()[:2], 2, SamplingParams(max_new_tokens=6))
    assert whole(eng)


@pytest.mark.gpu
def test_native_status_ends_the_call():
    from mod_b200.ops import native as N

    eng = _engine("native", "cuda:0", fp32=False)
    p = SamplingParams(max_new_tokens=6)
    want = eng.generate_parallel(_prompts()[:2], 2, p)
    far = torch.tensor([10 ** 6], dtype=torch.int32, device="cuda")
    N.kv_copy_pages(eng.kv.k, eng.kv.v, far, far)       # reported, nothing copied
    with pytest.raises(RuntimeError, match="out of bounds"):
        eng.generate_parallel(_prompts()[:2], 2, p)
    assert whole(eng)
    assert eng.generate_parallel(_prompts()[:2], 2, p) == want


# ------------------------------------------------------------------ what the engine keeps
def test_prefix_cache_outlives_uneven_ends():
    ref = _engine().generate(_prompts(), SamplingParams(max_new_tokens=24))
    eos = ref[0][2]
    eng = _engine(prefix_caching=True)
    old = [[700 + i for i in range(40)], [800 + i for i in range(33)]]
    want = eng.generate(old, SamplingParams(max_new_tokens=4))
    held = dict(eng.blocks.cache)
    assert len(held) >= 4
    got = eng.generate_parallel(_prompts(), 3, SamplingParams(max_new_tokens=24, eos_token_id=eos))
    assert [g[0] for g in got] == [r[:r.index(eos) + 1] if eos in r else r for r in ref]
    assert all(eng.blocks.cache.get(h) == b for h, b in held.items())
    hits = eng.blocks.hits
    assert eng.generate(old, SamplingParams(max_new_tokens=4)) == want
    assert eng.blocks.hits - hits == 2 + 2 and whole(eng)


def test_compact_counts_sixteen_tokens_a_block_whatever_its_size():
    from mod_b200.config import get_preset
    from mod_b200.engine.kv_cache import KVCache

    for bs in (4, 16, 32):
        kv = KVCache(get_preset("tiny-dense"), 12, "cpu", dtype=torch.float32, block_size=bs)
        for c in (*kv.k, *kv.v):
            c.copy_(torch.arange(12.0).view(12, 1, 1, 1).expand_as(c))
        tables = [[11, 2, 7, 9], [11, 5, 1]]
        remap, live = kv.compact(tables)
        assert live == 6 and {remap[b] for t in tables for b in t} == set(range(6))
        for c in (*kv.k, *kv.v):
            assert all((c[remap[b]] == b).all() for t in tables for b in t)


# ------------------------------------------------------------------ arguments
@pytest.mark.parametrize("n", [0, -1, -2, -17, 16, 100])
def test_counts_out_of_range_are_refused(n):
    with pytest.raises(ValueError, match="n ="):
        _engine().generate_parallel([[1, 2, 3]], n, SamplingParams(max_new_tokens=4))


# ------------------------------------------------------------------ little room
def test_drafts_take_what_the_next_tokens_leave(monkeypatch):
    from mod_b200.engine import parallel_sampling as M
    from mod_b200.engine.sequence import Sequence, SeqStatus

    eng = _engine(num_blocks=3)
    s = ParallelSampler(eng)
    s._seed(SamplingParams())
    params = SamplingParams(max_new_tokens=20)
    p = Sequence(prompt=list(range(1, 15)), params=params)
    assert eng.blocks.allocate(p, p.length)
    eng.runner.prefill([p], [p.length])
    a, b = Sequence(prompt=p.prompt, params=params), Sequence(prompt=p.prompt, params=params)
    eng.kv.copy_pages(eng.blocks.fork(p, a) + eng.blocks.fork(p, b))
    eng.blocks.release(p)
    a.output, b.output = [7], [7, 8, 9]           # b's last token needs the one free block, a's drafts would like it
    a.status = b.status = SeqStatus.RUNNING
    monkeypatch.setattr(M, "ngram_propose", lambda tokens, room, *n: [5] * room)
    s._step([[a, b]], [0])
    assert len(a.output) == 2 and len(b.blocks) == 2 and len(a.blocks) == 1
    assert s.stats.drafted > 0                     # b drafted into the rest of its block


@pytest.mark.parametrize("caching", [False, True])
@pytest.mark.parametrize("blocks", [5, 6, 8, 11, 20])
def test_prompts_wait_for_blocks(blocks, caching):
    # 40 tokens: two full blocks and one that is copied for each of two continuations; 8 more tokens fit the copies
    P = [[(31 * i + 7 * j) % 500 + 1 for j in range(40)] for i in range(5)]
    params = SamplingParams(max_new_tokens=8)
    ref = _engine(num_blocks=blocks).generate(P, params)
    eng = _engine(num_blocks=blocks, prefix_caching=caching)
    assert eng.generate_parallel(P, 2, params) == [[r] * 2 for r in ref]
    assert whole(eng)


def test_prompts_wait_for_places():
    P = [[(31 * i + 7 * j) % 500 + 1 for j in range(20)] for i in range(7)]
    params = SamplingParams(max_new_tokens=6)
    ref = _engine().generate(P, params)
    for n in (1, 5, 7, 8, 15):    # a batch of 16
        eng = _engine()
        assert eng.generate_parallel(P, n, params) == [[r] * n for r in ref]
        assert whole(eng)


@pytest.mark.parametrize("blocks", [7, 9])
def test_other_requests_hold_the_blocks(blocks):
    # two requests are under way when the call comes; it needs five blocks, and they are run until these are free
    P = [[(31 * i + 7 * j) % 500 + 1 for j in range(40)] for i in range(3)]
    params = SamplingParams(max_new_tokens=8)
    ref = _engine().generate(P, params)
    eng = _engine(num_blocks=blocks)
    ids = [eng.add_request(p, params) for p in P[:2]]
    eng.step()
    assert eng.scheduler.running
    assert eng.generate_parallel(P[2:], 2, params) == [[ref[2]] * 2]
    while eng.has_unfinished():
        eng.step()
    assert [eng.seqs[i].output for i in ids] == ref[:2] and whole(eng)


@pytest.mark.parametrize("caching", [False, True])
@pytest.mark.parametrize("drafts", [0, 3])
@pytest.mark.parametrize("blocks", range(8, 22))
def test_sequences_that_outgrow_the_pool_come_back(blocks, drafts, caching):
    # what generate() does with the same sequences one beside another in the same pool
    P, params = _prompts()[:3], SamplingParams(max_new_tokens=20)
    ref = _engine(num_blocks=blocks).generate([p for p in P for _ in range(3)], params)
    eng = _engine(num_blocks=blocks, prefix_caching=caching)
    s = ParallelSampler(eng, drafts=drafts)
    assert [x for g in s.generate(P, 3, params) for x in g] == ref
    assert whole(eng)


def test_each_sequence_is_computed_again_once_at_most():
    P, params = _prompts()[:3], SamplingParams(max_new_tokens=60)
    ref = _engine().generate(P, params)
    eng = _engine(num_blocks=14)
    s = ParallelSampler(eng)
    back = []
    fork = eng.blocks.fork
    eng.blocks.fork = lambda p, c, *n: (back.append(c.req_id) if c.output else None) or fork(p, c, *n)
    assert s.generate(P, 4, params) == [[r] * 4 for r in ref]
    assert back and len(set(back)) == len(back) and eng.scheduler.num_preempted >= len(back)


def test_one_sequence_that_does_not_fit_is_refused():
    # 36 + 63 cached tokens take 7 blocks
    P, params = [_prompts()[0]], SamplingParams(max_new_tokens=64)
    for blocks in (5, 6):
        eng = _engine(num_blocks=blocks)
        with pytest.raises(RuntimeError, match="exhausted"):
            eng.generate_parallel(P, 2, params)
        assert whole(eng)
    eng = _engine(num_blocks=7)
    assert eng.generate_parallel(P, 2, params) == [_engine().generate(P, params) * 2] and whole(eng)


def test_growth_beside_other_requests():
    P, params = _prompts()[:3], SamplingParams(max_new_tokens=40)
    ref = _engine().generate(P, params)
    eng = _engine(num_blocks=11)
    rid = eng.add_request(P[2], params)
    eng.step()
    assert eng.generate_parallel(P[:2], 2, params) == [[r] * 2 for r in ref[:2]]
    while eng.has_unfinished():
        eng.step()
    assert eng.seqs[rid].output == ref[2] and whole(eng)


# ------------------------------------------------------------------ seeds
@pytest.mark.parametrize("drafts", [0, 4])
def test_seeded_continuations_do_not_depend_on_the_other_prompts(drafts):
    P, params = _prompts(), SamplingParams(max_new_tokens=16, temperature=0.9, seed=11)
    run = lambda prompts, n=3, **kw: ParallelSampler(_engine(**kw), drafts=drafts).generate(prompts, n, params)  # noqa: E731
    alone = [run([p])[0] for p in P]
    assert run(P) == alone and run(P[::-1]) == alone[::-1] and run([P[2], P[0]]) == [alone[2], alone[0]]
    assert [g[:2] for g in alone] == run(P, 2)            # nor on how many there are
    assert len({tuple(x) for g in alone for x in g}) == len(P) * 3
    # a call on the same engine repeats it, one with another seed does not
    s = ParallelSampler(_engine(), drafts=drafts)
    assert s.generate(P[:1], 3, params) == s.generate(P[:1], 3, params) == alone[:1] and not s.gens
    assert s.generate(P[:1], 3, SamplingParams(max_new_tokens=16, temperature=0.9, seed=12)) != alone[:1]


@pytest.mark.gpu
def test_native_seeded_continuations_do_not_depend_on_the_other_prompts():
    # bf16 rounds with the batch a prompt is computed in, so that a later token may differ by that alone: the first one,
    # drawn from the prompt's own logits, has to be the same for most, and every one for the same call
    P, params = _prompts(), SamplingParams(max_new_tokens=8, temperature=0.9, seed=11)
    run = lambda prompts: _engine("native", "cuda:0", fp32=False).generate_parallel(prompts, 4, params)  # noqa: E731
    a, b = run(P), run(P[::-1])[::-1]
    first = [x[0] == y[0] for g, h in zip(a, b) for x, y in zip(g, h)]
    assert sum(first) >= len(first) - 1 and run(P) == a


def test_unseeded_continuations_differ():
    params = SamplingParams(max_new_tokens=12, temperature=1.0)
    s = ParallelSampler(_engine())
    got = [x for _ in range(2) for g in s.generate(_prompts()[:2], 4, params) for x in g]
    assert len({tuple(x) for x in got}) > 12


def test_sampled_sequences_that_come_back_go_on_as_they_were():
    # sampled tokens do not depend on when a sequence had blocks, without drafts
    P, params = _prompts()[:3], SamplingParams(max_new_tokens=30, temperature=1.0, top_k=40, seed=9)
    want = ParallelSampler(_engine(), drafts=0).generate(P, 3, params)
    small = _engine(num_blocks=9)
    got = ParallelSampler(small, drafts=0).generate(P, 3, params)
    assert small.scheduler.num_preempted > 0 and whole(small)
    assert all(len(x) == 30 for g in got for x in g) and got == want


@pytest.mark.gpu
@pytest.mark.parametrize("caching", [False, True])
def test_native_sequences_that_outgrow_the_pool_come_back(caching):
    # the computed-again step has as many query tokens as a sequence had emitted, over the shared-prefix kernels
    from mod_b200.engine.sequence import Sequence

    P, params = _prompts(), SamplingParams(max_new_tokens=90)
    ref = _engine("native", "cuda:0", fp32=False).generate(P, params)
    eng = _engine("native", "cuda:0", fp32=False, num_blocks=19, prefix_caching=caching)
    got = eng.generate_parallel(P, 3, params)
    assert eng.scheduler.num_preempted > 0 and whole(eng)
    # Where a continuation leaves the greedy one, the two tokens' logits have to tie, within two bf16 roundings (2^-8 each)
    # in each of the two paths.
    for prompt, r, g in zip(P, ref, got):
        for x in g:
            assert len(x) == 90
            k = next((i for i in range(90) if x[i] != r[i]), None)
            if k is None:
                continue
            q = Sequence(prompt=prompt + r[:k], params=SamplingParams())
            assert eng.blocks.allocate(q, q.length)
            logits = eng.runner.prefill([q], [q.length - q.num_cached], return_logits=True)[0]
            eng.blocks.release(q)
            top = float(logits.max())
            assert min(float(logits[x[k]]), float(logits[r[k]])) >= top - 2 ** -6 * float(logits.abs().max()), (k, x, r)
